// Selection of the best continuations of beams over a vocabulary.
//
// Candidate (k, v) of a batch row is worth score_k + x_kv - log sum_w exp(x_kw).
// Within a beam the order is that of the logits, so one pass over the logits
// finds a beam's sum and its n best tokens; the second kernel turns the few that
// are left into candidates and takes the n best of all beams.
#include "kf_common.cuh"
#include "kv8_common.cuh"

namespace kf {

constexpr int BEAM_THREADS = 256;
constexpr int BEAM_MAX = 128;    // candidates of a call
constexpr int BEAM_CAP = 4096;   // keys that the first kernel's list holds
constexpr int BEAM_JOIN_CAP = 2048;
constexpr float BEAM_LOG2E = 1.4426950408889634f;

struct BeamWork {
  uint64_t* key;   // [rows][slices][n]: a logit in order, then the complement of its index; 0: none
  float* top;      // [rows][slices]
  double* sum;     // [rows][slices]: of exp(x - top)
  int slices;
  int64_t slice;   // tokens of a slice
};

// A number as bits in its order; -0 and +0 are one.
__device__ __forceinline__ uint32_t beam_order(float x) {
  const uint32_t u = __float_as_uint(__fadd_rn(x, 0.f));
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float beam_value(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

// A candidate of the second kernel: its fp64 value as an integer in the same order,
// then the complements of beam and token. 0: none.
struct alignas(16) BeamKey {
  uint64_t c;
  uint64_t at;
};
__device__ __forceinline__ uint64_t beam_order(double x) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x + 0.0));  // (-0 and +0 are one)
  return (u >> 63) ? ~u : (u | (1ull << 63));
}
__device__ __forceinline__ double beam_value(uint64_t o) {
  return __longlong_as_double(static_cast<long long>((o >> 63) ? (o ^ (1ull << 63)) : ~o));
}
__device__ __forceinline__ bool beam_before(const BeamKey& a, const BeamKey& b) {
  return a.c > b.c || (a.c == b.c && a.at > b.at);
}
__device__ __forceinline__ bool beam_before(uint64_t a, uint64_t b) { return a > b; }
__device__ __forceinline__ void beam_none(uint64_t& k) { k = 0; }
__device__ __forceinline__ void beam_none(BeamKey& k) { k.c = k.at = 0; }

// Sorts the first `count` of a list in shared memory, best first. The list has
// room up to the next power of two. All threads of the CTA.
template <class Key>
__device__ void beam_sort(Key* list, int count) {
  int size = 2;
  while (size < count) size <<= 1;
  for (int i = count + threadIdx.x; i < size; i += BEAM_THREADS) beam_none(list[i]);
  __syncthreads();
  for (int run = 2; run <= size; run <<= 1)
    for (int step = run >> 1; step; step >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += BEAM_THREADS) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const Key a = list[lo], b = list[hi];
        const bool up = (lo & run) == 0;
        if (up ? beam_before(b, a) : beam_before(a, b)) {
          list[lo] = b;
          list[hi] = a;
        }
      }
      __syncthreads();
    }
}

// The n best of the first `count` keys of a list in shared memory, best first, by
// put(place, key): every key counts those before it, which for a few hundred keys
// is far shorter than a sort's chain of barriers. All threads of the CTA; `list` is
// read only after a barrier of the caller's. Many keys are sorted.
constexpr int BEAM_COUNTED = 512;
template <class Key, class Put>
__device__ __forceinline__ void beam_best(Key* list, int count, int n, Put&& put) {
  if (count > BEAM_COUNTED) {
    beam_sort(list, count);
    for (int i = threadIdx.x; i < min(n, count); i += BEAM_THREADS) put(i, list[i]);
    return;
  }
  for (int i = threadIdx.x; i < count; i += BEAM_THREADS) {
    const Key mine = list[i];
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < count; ++j) place += beam_before(list[j], mine) ? 1 : 0;
    if (place < n) put(place, mine);
  }
}

// ---------------------------------------------------------------- one pass over the logits
//
// One CTA = a slice of a beam's vocabulary, 4 x 16 bytes of logits a thread in
// flight. The first round (up to 4096 or 8192 tokens) gives the threads' largest
// logits; the n-th largest of those is a bound that at least n tokens reach, so what
// is below it is passed over with one comparison for each 16 bytes, and the list
// of the others stays short without any barrier in the loop. Where it does not
// (many equal logits, or logits that grow along the slice), the slice is read
// again in small rounds that cut the list as it fills.
// What bounds it: latency. 64 x 8 rows of 128000 bf16 logits take 62 us for 124 MB (floor
// 19; with a barrier and a list of all candidates in every round 138): a quarter
// of the copy rate, 58 % of the issue slots while an SM has work (17 instructions
// a logit: four and an exponential of its sum, the rest the appends of 16-byte runs
// with a token above the bound, 2 % of the runs but every second one of a warp, with 22
// of 32 lanes active) and 35 % of the exponentials' pipe. Six warps a scheduler
// wait 2.5 cycles an issue on fixed latencies and 2.4 on loads: a round's are asked for
// when the last one is summed, not before. 512 CTAs on 148 SMs leave some with three
// of four. 24 x 8 rows of 50021 fp32 logits, 35 MB, about 20 us.

template <int DT>
__device__ __forceinline__ void beam_load(const void* logits, int64_t base, int64_t i, int64_t last,
                                          bool vec, uint4& v) {
  constexpr int N = KV8Type<DT>::N;
  if (i + N <= last) {
    v = KV8Type<DT>::load(logits, base + i, vec);
    return;
  }
  // the end: what is not there is -inf
  uint32_t w[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if constexpr (DT == KF_DT_F32) {
      w[u] = i + u < last ? static_cast<const uint32_t*>(logits)[base + i + u] : 0xff800000u;
    } else {
      constexpr uint32_t none = DT == KF_DT_BF16 ? 0xff80u : 0xfc00u;
      const uint16_t* q = static_cast<const uint16_t*>(logits) + base;
      const int64_t j = i + 2 * u;
      w[u] = (j < last ? q[j] : none) | ((j + 1 < last ? q[j + 1] : none) << 16);
    }
  }
  v = make_uint4(w[0], w[1], w[2], w[3]);
}

// The largest number of a 16-byte run (NaN if it has none), and its u-th one.
template <int DT>
struct BeamMax {
  __device__ __forceinline__ static float of(const uint4& v) {
    if constexpr (DT == KF_DT_F32) {
      return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                   fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    } else if constexpr (DT == KF_DT_BF16) {
      auto h = [](const uint32_t& w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
      const __nv_bfloat162 m = __hmax2(__hmax2(h(v.x), h(v.y)), __hmax2(h(v.z), h(v.w)));
      return fmaxf(__low2float(m), __high2float(m));
    } else {
      auto h = [](const uint32_t& w) { return *reinterpret_cast<const __half2*>(&w); };
      const __half2 m = __hmax2(__hmax2(h(v.x), h(v.y)), __hmax2(h(v.z), h(v.w)));
      return fmaxf(__low2float(m), __high2float(m));
    }
  }
  __device__ __forceinline__ static float at(const uint4& v, int u) {
    const int i = DT == KF_DT_F32 ? u : u >> 1;
    const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
    if constexpr (DT == KF_DT_F32) return __uint_as_float(w);
    const uint32_t h = (u & 1) ? w >> 16 : w & 0xffffu;
    if constexpr (DT == KF_DT_BF16) return __uint_as_float(h << 16);
    return __half2float(__ushort_as_half(static_cast<uint16_t>(h)));
  }
};

// Keys of the n best tokens of a slice, at the front of the list; how many.
template <int DT>
__device__ __noinline__ int beam_careful(uint64_t* list, int* s_count, const void* logits,
                                         int64_t base, int64_t first, int64_t last, bool vec, int n) {
  constexpr int N = KV8Type<DT>::N;
  uint64_t cut = 0;   // keys up to it are out: n better ones are known
  __syncthreads();
  if (threadIdx.x == 0) *s_count = 0;
  __syncthreads();
  for (int64_t at = first; at < last; at += N * BEAM_THREADS) {
    const int64_t i = at + threadIdx.x * N;
    uint4 v;
    float x[N];
    beam_load<DT>(logits, base, i, last, vec, v);
    KV8Type<DT>::values(v, x);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (!(x[u] > -INFINITY)) continue;   // NaN among them
      const uint64_t key = static_cast<uint64_t>(beam_order(x[u])) << 32 |
                           (0xffffffffu - static_cast<uint32_t>(i + u));
      if (key > cut) list[atomicAdd(s_count, 1)] = key;
    }
    __syncthreads();
    const int count = *s_count;
    if (count > BEAM_CAP - N * BEAM_THREADS) {
      beam_sort(list, count);
      cut = list[n - 1];
      if (threadIdx.x == 0) *s_count = n;
    }
    __syncthreads();
  }
  return *s_count;
}

template <int DT>
__global__ void __launch_bounds__(BEAM_THREADS, 4)
    beam_scan_kernel(const void* __restrict__ logits, int64_t l_sb, int64_t l_sk, int vec,
                     const uint8_t* __restrict__ ended, int64_t e_sb, int beams, int64_t vocab,
                     int n, BeamWork w) {
  constexpr int N = KV8Type<DT>::N, U = 4;
  __shared__ uint64_t list[BEAM_CAP];
  __shared__ __align__(16) uint32_t s_max[BEAM_THREADS];
  __shared__ uint32_t s_cut;
  __shared__ int s_count;
  __shared__ float s_top[BEAM_THREADS / 32];
  __shared__ double s_sum[BEAM_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.y;
  const int b = row / beams, k = row - b * beams;
  const int64_t spot = static_cast<int64_t>(row) * w.slices + blockIdx.x;
  if (ended && ended[b * e_sb + k]) return;   // its candidate needs no logits
  const int64_t first = blockIdx.x * w.slice;
  const int64_t last = first + w.slice < vocab ? first + w.slice : vocab;
  const int64_t base = b * l_sb + k * l_sk;
  float top = -INFINITY;
  uint64_t sum = f2_pack(0.f, 0.f);  // two sums
  float cut = -INFINITY;   // logits below it are out, and those equal to it after the first round
  if (tid == 0) s_count = 0;   // (a barrier comes before it is used)
  // The n-th largest of the threads' numbers: at least n logits are not below it.
  // -inf if there are fewer.
  auto bound = [&](float most) -> float {
    const uint32_t mine = most > -INFINITY ? beam_order(most) : 0u;
    s_max[tid] = mine;
    if (tid == 0) s_cut = 0xffffffffu;
    __syncthreads();
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < BEAM_THREADS; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(s_max + j);
      above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
    }
    if (above < n) atomicMin(&s_cut, mine);
    __syncthreads();
    return s_cut ? beam_value(s_cut) : -INFINITY;
  };
  float best = -INFINITY;  // this thread's largest logit
  // `apart`: the thread's logits are BEAM_THREADS tokens apart, not runs of N.
  auto round = [&](const uint4 (&v)[U], int64_t at, bool begin, bool apart) {
    float m[U];
#pragma unroll
    for (int r = 0; r < U; ++r) m[r] = BeamMax<DT>::of(v[r]);
    float most = m[0];
#pragma unroll
    for (int r = 1; r < U; ++r) most = fmaxf(most, m[r]);
    if (begin) cut = bound(most);
    best = fmaxf(best, most);
    if (most > top) {
      const float a = fast_exp2((top - most) * BEAM_LOG2E);
      sum = f2_mul(sum, f2_pack(a, a));
      top = most;
    }
    // (x - top first: the fused x log2 e - top log2 e would leave the rounding of the
    // second product in the exponent, which at logits of 10^4 is 2^-10)
    const float ref = top == -INFINITY ? 0.f : -top;
#pragma unroll
    for (int r = 0; r < U; ++r) {
      float x[N];
      KV8Type<DT>::values(v[r], x);
#pragma unroll
      for (int u = 0; u < N; u += 2) {
        float e, f;
        f2_unpack(f2_mul(f2_add(f2_pack(x[u], x[u + 1]), f2_pack(ref, ref)),
                         f2_pack(BEAM_LOG2E, BEAM_LOG2E)), e, f);
        sum = f2_add(sum, f2_pack(fast_exp2(e), fast_exp2(f)));
      }
      if (begin ? m[r] >= cut : m[r] > cut) {
        const uint32_t i = static_cast<uint32_t>(at + r * BEAM_THREADS * N + (apart ? tid : tid * N));
        const uint32_t next = apart ? BEAM_THREADS : 1;
#pragma unroll
        for (int u = 0; u < N; ++u)
          if (x[u] > -INFINITY && (begin ? x[u] >= cut : x[u] > cut)) {
            const int to = atomicAdd(&s_count, 1);
            if (to < BEAM_CAP)
              list[to] = static_cast<uint64_t>(beam_order(x[u])) << 32 | (0xffffffffu - (i + u * next));
          }
      }
      __syncwarp();   // (lanes that went that way would go on alone: five of 32 active)
    }
  };
  constexpr int64_t ROUND = U * N * BEAM_THREADS;
#pragma unroll 1
  for (int64_t at = first; at < last; at += ROUND) {
    uint4 v[U];
    const bool apart = !vec && at + ROUND <= last;
    if (apart) {
      // Rows that are not aligned (an odd vocabulary): neighbours load neighbours.
      constexpr int SIZE = DT == KF_DT_F32 ? 4 : 2;
      const uint8_t* p = static_cast<const uint8_t*>(logits) + (base + at + tid) * SIZE;
#pragma unroll
      for (int r = 0; r < U; ++r) {
        uint32_t x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if constexpr (DT == KF_DT_F32) {
            x[u] = __ldg(reinterpret_cast<const uint32_t*>(p) + (r * N + u) * BEAM_THREADS);
          } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + (r * N + 2 * u) * BEAM_THREADS;
            x[u] = __ldg(h) | (static_cast<uint32_t>(__ldg(h + BEAM_THREADS)) << 16);
          }
        }
        v[r] = make_uint4(x[0], x[1], x[2], x[3]);
      }
    } else if (vec && at + ROUND <= last) {
      const uint4* p = reinterpret_cast<const uint4*>(
          static_cast<const uint8_t*>(logits) + (base + at) * (DT == KF_DT_F32 ? 4 : 2)) + tid;
#pragma unroll
      for (int r = 0; r < U; ++r) v[r] = __ldg(p + r * BEAM_THREADS);
    } else {
#pragma unroll 1
      for (int r = 0; r < U; ++r) {
        uint4 one;
        beam_load<DT>(logits, base, at + (r * BEAM_THREADS + tid) * N, last, vec != 0, one);
#pragma unroll
        for (int q = 0; q < U; ++q)
          if (q == r) v[q] = one;
      }
    }
    round(v, at, at == first, apart);
  }
  __syncthreads();
  int count = s_count;
  uint64_t* from = list;
  if (count > BEAM_CAP) {
    count = beam_careful<DT>(list, &s_count, logits, base, first, last, vec != 0, n);
  } else if (count > 2 * n) {
    // By now a better bound is known: what reaches it moves behind the list.
    const float last_cut = bound(best);
    if (tid == 0) s_count = 0;
    __syncthreads();
    const uint64_t least = static_cast<uint64_t>(beam_order(last_cut)) << 32;
    const int room = min(BEAM_CAP - count, BEAM_COUNTED);   // (what is sorted needs more)
    from = list + count;
    for (int i = tid; i < count; i += BEAM_THREADS)
      if (list[i] >= least) {
        const int to = atomicAdd(&s_count, 1);
        if (to < room) from[to] = list[i];
      }
    __syncthreads();
    if (s_count <= room)
      count = s_count;
    else
      from = list;       // too many to move: all of them, then
  }
  uint64_t* out = w.key + spot * n;
  beam_best(from, count, n, [&](int place, uint64_t key) { out[place] = key; });
  for (int i = count + tid; i < n; i += BEAM_THREADS) out[i] = 0;
  // the slice's sum
  float m = top;
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (lane == 0) s_top[warp] = m;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < BEAM_THREADS / 32; ++u) m = fmaxf(m, s_top[u]);
  // (a thread that saw no number has a sum of 0, or NaN)
  float s0, s1;
  f2_unpack(sum, s0, s1);
  double s = static_cast<double>(s0) + static_cast<double>(s1);
  if (top != -INFINITY) s *= fast_exp2((top - m) * BEAM_LOG2E);
#pragma unroll
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (lane == 0) s_sum[warp] = s;
  __syncthreads();
  if (tid == 0) {
    for (int u = 1; u < BEAM_THREADS / 32; ++u) s += s_sum[u];
    w.top[spot] = m;
    w.sum[spot] = s;
  }
}

// ---------------------------------------------------------------- the best of all beams
//
// One CTA a batch row: the beams' sums, a warp each, then their keys as candidates.
// Latency is what it costs, 10 to 16 us when its code is fetched for the first time.
// The slices' lists are in order, so the n-th best of their first ones bounds the
// answer, and few candidates are left to compare.

__global__ void __launch_bounds__(BEAM_THREADS)
    beam_join_kernel(const float* __restrict__ scores, int64_t s_sb,
                     const uint8_t* __restrict__ ended, int64_t e_sb, int beams, int n, int32_t pad,
                     float* __restrict__ out_score, int32_t* __restrict__ out_beam,
                     int32_t* __restrict__ out_token, BeamWork w) {
  __shared__ BeamKey list[BEAM_JOIN_CAP];
  __shared__ BeamKey s_cut;
  __shared__ double s_lse[1024];   // of a beam; of an ended one not used
  __shared__ float s_score[1024];
  __shared__ uint8_t s_ended[1024];
  __shared__ int s_count;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x;
  for (int k = warp; k < beams; k += BEAM_THREADS / 32) {
    const int64_t spot = (static_cast<int64_t>(b) * beams + k) * w.slices;
    const bool end = ended && ended[b * e_sb + k];
    if (lane == 0) {
      s_ended[k] = end;
      s_score[k] = scores[b * s_sb + k];
    }
    if (end) continue;
    float m = -INFINITY;
    for (int i = lane; i < w.slices; i += 32) m = fmaxf(m, w.top[spot + i]);
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    double s = 0.0;
    for (int i = lane; i < w.slices; i += 32) {
      const double part = w.sum[spot + i];
      if (part != 0.0) s += part * fast_exp2((w.top[spot + i] - m) * BEAM_LOG2E);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0) s_lse[k] = m + log(s);
  }
  if (tid == 0) {
    s_count = 0;
    beam_none(s_cut);
  }
  __syncthreads();
  const int64_t per = static_cast<int64_t>(w.slices) * n;
  const int64_t all = beams * per;
  // Entry i of the row's lists as a candidate; false: it is none.
  auto candidate = [&](int64_t i, BeamKey& c) -> bool {
    const int k = static_cast<int>(i / per);
    double x;
    if (s_ended[k]) {
      if (i != k * per) return false;
      x = s_score[k];
      c.at = ~(static_cast<uint64_t>(k) << 32 | static_cast<uint32_t>(pad));
    } else {
      const uint64_t key = w.key[static_cast<int64_t>(b) * all + i];
      if (!key) return false;
      x = (static_cast<double>(beam_value(static_cast<uint32_t>(key >> 32))) - s_lse[k]) + s_score[k];
      c.at = ~(static_cast<uint64_t>(k) << 32 | (0xffffffffu - static_cast<uint32_t>(key)));
    }
    if (!(x > -INFINITY)) return false;
    c.c = beam_order(x);
    return true;
  };
  const int lists = beams * w.slices;
  const int depth = (n + lists - 1) / lists;   // first entries of every list: at least n
  if (all > 2 * BEAM_MAX && lists * depth <= BEAM_COUNTED) {
    for (int i = tid; i < lists * depth; i += BEAM_THREADS) {
      BeamKey c;
      if (candidate(static_cast<int64_t>(i / depth) * n + i % depth, c))
        list[atomicAdd(&s_count, 1)] = c;
    }
    __syncthreads();
    const int count = s_count;
    beam_best(list, count, n, [&](int place, const BeamKey& c) {
      if (place == n - 1) s_cut = c;
    });
    __syncthreads();
    if (tid == 0) s_count = 0;
    __syncthreads();
  }
  BeamKey cut = s_cut;   // candidates after it are out
  for (int64_t at = 0; at < all; at += BEAM_THREADS) {
    const int64_t i = at + tid;
    BeamKey c;
    if (i < all && candidate(i, c) && !beam_before(cut, c)) list[atomicAdd(&s_count, 1)] = c;
    if (all <= BEAM_JOIN_CAP) continue;
    __syncthreads();
    const int count = s_count;
    if (count > BEAM_JOIN_CAP - BEAM_THREADS) {
      beam_sort(list, count);
      cut = list[n - 1];
      if (tid == 0) s_count = n;
    }
    __syncthreads();
  }
  __syncthreads();
  const int count = s_count;
  const int64_t o = static_cast<int64_t>(b) * n;
  beam_best(list, count, n, [&](int place, const BeamKey& c) {
    out_score[o + place] = static_cast<float>(beam_value(c.c));
    out_beam[o + place] = static_cast<int32_t>(~c.at >> 32);
    out_token[o + place] = static_cast<int32_t>(static_cast<uint32_t>(~c.at));
  });
  for (int i = count + tid; i < n; i += BEAM_THREADS) {
    out_score[o + i] = -INFINITY;
    out_beam[o + i] = -1;
    out_token[o + i] = -1;
  }
}

// ---------------------------------------------------------------- host

static int beam_check(const char* what, int64_t batch, int64_t beams, int64_t vocab, int64_t n) {
  if (batch < 0 || beams <= 0 || vocab <= 0 || n <= 0) {
    set_last_error("%s: needs batch >= 0 and beams, vocab and n of at least 1", what);
    return KF_E_INVALID;
  }
  if (n > BEAM_MAX || beams > 1024 || vocab > INT32_MAX || batch * beams > 65535) {
    set_last_error("%s: needs n <= %d, beams <= 1024, vocab < 2^31 and batch * beams <= 65535", what,
                   BEAM_MAX);
    return KF_E_UNSUPPORTED;
  }
  return KF_OK;
}

static int64_t beam_carve(int64_t batch, int64_t beams, int64_t vocab, int64_t n, uint8_t* base,
                          BeamWork* w) {
  const int64_t rows = batch * beams;
  // One wave of four CTAs an SM; slices of at least a round of 4096 tokens.
  int64_t slices = rows ? sm_count() * 4 / rows : 1;
  const int64_t most = (vocab + 4095) / 4096;
  if (slices > most) slices = most;
  if (slices < 1) slices = 1;
  w->slice = ((vocab + slices - 1) / slices + 7) / 8 * 8;
  w->slices = static_cast<int>((vocab + w->slice - 1) / w->slice);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    uint8_t* p = base + at;
    at += (bytes + 15) / 16 * 16;
    return p;
  };
  w->key = reinterpret_cast<uint64_t*>(take(rows * w->slices * n * 8));
  w->sum = reinterpret_cast<double*>(take(rows * w->slices * 8));
  w->top = reinterpret_cast<float*>(take(rows * w->slices * 4));
  return at;
}

}  // namespace kf

using namespace kf;

extern "C" int64_t kf_beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab,
                                                  int64_t n) {
  if (beam_check("kf_beam_select_workspace_bytes", batch, beams, vocab, n)) return -1;
  if (batch == 0) return 0;
  BeamWork w;
  return beam_carve(batch, beams, vocab, n, nullptr, &w);
}

extern "C" int kf_beam_select(const void* logits, int64_t l_sb, int64_t l_sk, int dtype,
                              const float* scores, int64_t s_sb, const uint8_t* ended, int64_t e_sb,
                              int64_t batch, int64_t beams, int64_t vocab, int64_t n, int32_t pad,
                              float* out_score, int32_t* out_beam, int32_t* out_token,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "kf_beam_select";
  int rc = beam_check(what, batch, beams, vocab, n);
  if (!rc) rc = kv8_dtype(what, dtype);
  if (rc) return rc;
  if (batch == 0) return KF_OK;
  if (!logits || !scores || !out_score || !out_beam || !out_token || pad < 0) {
    set_last_error("%s: pointers must not be null, and pad not negative", what);
    return KF_E_INVALID;
  }
  BeamWork w;
  const int64_t need = beam_carve(batch, beams, vocab, n, static_cast<uint8_t*>(workspace), &w);
  if (!workspace || workspace_bytes < need || !kv8_aligned(workspace, 16)) {
    set_last_error("%s: needs a 16-byte aligned workspace of %lld bytes", what, (long long)need);
    return KF_E_INVALID;
  }
  const int64_t per = 16 / dtype_size(dtype);
  const int vec = kv8_aligned(logits, 16) && l_sb % per == 0 && l_sk % per == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto scan = dtype == KF_DT_F32    ? beam_scan_kernel<KF_DT_F32>
              : dtype == KF_DT_BF16 ? beam_scan_kernel<KF_DT_BF16>
                                    : beam_scan_kernel<KF_DT_F16>;
  cudaError_t e = launch_chained(
      scan, dim3(static_cast<unsigned>(w.slices), static_cast<unsigned>(batch * beams)),
      dim3(BEAM_THREADS), 0, st, logits, l_sb, l_sk, vec, ended, e_sb, static_cast<int>(beams), vocab,
      static_cast<int>(n), w);
  if (e != cudaSuccess) return cuda_status(e, "kf_beam_select scan launch");
  e = launch_chained(beam_join_kernel, dim3(static_cast<unsigned>(batch)), dim3(BEAM_THREADS), 0, st,
                     scores, s_sb, ended, e_sb, static_cast<int>(beams), static_cast<int>(n), pad,
                     out_score, out_beam, out_token, w);
  return cuda_status(e, "kf_beam_select join launch");
}
