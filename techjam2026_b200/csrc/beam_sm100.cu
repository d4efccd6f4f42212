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

// A candidate of the second kernel.
struct alignas(16) BeamKey {
  double c;
  uint64_t at;     // beam << 32 | token
};
__device__ __forceinline__ bool beam_before(const BeamKey& a, const BeamKey& b) {
  return a.c > b.c || (a.c == b.c && a.at < b.at);
}
__device__ __forceinline__ bool beam_before(uint64_t a, uint64_t b) { return a > b; }
__device__ __forceinline__ void beam_none(uint64_t& k) { k = 0; }
__device__ __forceinline__ void beam_none(BeamKey& k) {
  k.c = -INFINITY;
  k.at = ~0ull;
}

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
// Bound by memory, and by the exponentials for 16-bit logits (16 a clock and SM).

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
  constexpr float LOG2E = 1.4426950408889634f;
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
  float top = -INFINITY, sum = 0.f;
  float cut = -INFINITY;   // logits below it are out, and those equal to it after the first round
  if (tid == 0) {
    s_count = 0;
    s_cut = 0;
  }
  for (int64_t at = first; at < last; at += U * N * BEAM_THREADS) {
    uint4 v[U];
#pragma unroll
    for (int r = 0; r < U; ++r)
      beam_load<DT>(logits, base, at + (r * BEAM_THREADS + tid) * N, last, vec != 0, v[r]);
    float m[U];
#pragma unroll
    for (int r = 0; r < U; ++r) {
      float x[N];
      KV8Type<DT>::values(v[r], x);
      m[r] = x[0];
#pragma unroll
      for (int u = 1; u < N; ++u) m[r] = fmaxf(m[r], x[u]);
    }
    float most = m[0];
#pragma unroll
    for (int r = 1; r < U; ++r) most = fmaxf(most, m[r]);
    if (at == first) {
      // (a thread without a number has 0, below every number's order)
      const uint32_t mine = most > -INFINITY ? beam_order(most) : 0u;
      s_max[tid] = mine;
      __syncthreads();
      int before = 0;
#pragma unroll 8
      for (int j = 0; j < BEAM_THREADS; j += 4) {
        const uint4 o = *reinterpret_cast<const uint4*>(s_max + j);
        before += (o.x > mine || (o.x == mine && j < tid)) + (o.y > mine || (o.y == mine && j + 1 < tid)) +
                  (o.z > mine || (o.z == mine && j + 2 < tid)) + (o.w > mine || (o.w == mine && j + 3 < tid));
      }
      if (before == n - 1) s_cut = mine;
      __syncthreads();
      if (s_cut) cut = beam_value(s_cut);
    }
    if (most > top) {
      sum *= fast_exp2((top - most) * LOG2E);
      top = most;
    }
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int r = 0; r < U; ++r) {
      float x[N];
      KV8Type<DT>::values(v[r], x);
#pragma unroll
      for (int u = 0; u < N; ++u) sum += fast_exp2((x[u] - ref) * LOG2E);
      if (at == first ? m[r] >= cut : m[r] > cut) {
        const uint32_t i = static_cast<uint32_t>(at + (r * BEAM_THREADS + tid) * N);
#pragma unroll
        for (int u = 0; u < N; ++u)
          if (x[u] > -INFINITY && (at == first ? x[u] >= cut : x[u] > cut)) {
            const int to = atomicAdd(&s_count, 1);
            if (to < BEAM_CAP)
              list[to] = static_cast<uint64_t>(beam_order(x[u])) << 32 | (0xffffffffu - (i + u));
          }
      }
    }
  }
  __syncthreads();
  int count = s_count;
  if (count > BEAM_CAP)
    count = beam_careful<DT>(list, &s_count, logits, base, first, last, vec != 0, n);
  uint64_t* out = w.key + spot * n;
  beam_best(list, count, n, [&](int place, uint64_t key) { out[place] = key; });
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
  double s = static_cast<double>(top == -INFINITY ? sum : sum * fast_exp2((top - m) * LOG2E));
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
// Latency is what it costs. The slices' lists are in order, so the n-th best of
// their first entries bounds the answer, and few candidates are left to compare.

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
      if (part != 0.0) s += part * exp(static_cast<double>(w.top[spot + i]) - m);
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
    if (s_ended[k]) {
      if (i != k * per) return false;
      c.c = s_score[k];
      c.at = static_cast<uint64_t>(k) << 32 | static_cast<uint32_t>(pad);
    } else {
      const uint64_t key = w.key[static_cast<int64_t>(b) * all + i];
      if (!key) return false;
      c.c = (static_cast<double>(beam_value(static_cast<uint32_t>(key >> 32))) - s_lse[k]) +
            s_score[k];
      c.at = static_cast<uint64_t>(k) << 32 | (0xffffffffu - static_cast<uint32_t>(key));
    }
    return c.c > -INFINITY;
  };
  const int64_t heads = static_cast<int64_t>(beams) * w.slices;
  if (all > BEAM_COUNTED && heads >= n && heads <= BEAM_COUNTED) {
    for (int64_t i = tid; i < heads; i += BEAM_THREADS) {
      BeamKey c;
      if (candidate(i * n, c)) list[atomicAdd(&s_count, 1)] = c;
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
    out_score[o + place] = static_cast<float>(c.c);
    out_beam[o + place] = static_cast<int32_t>(c.at >> 32);
    out_token[o + place] = static_cast<int32_t>(static_cast<uint32_t>(c.at));
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
