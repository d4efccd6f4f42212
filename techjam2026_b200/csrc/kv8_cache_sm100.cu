// Writing, reading and thinning the 8-bit key/value cache.
#include "kv8_common.cuh"

namespace kf {

// ---------------------------------------------------------------- append
//
// One CTA per (page a chunk can reach, kv head, sequence). It loads the page's
// new tokens of K and V as they are into registers (16 bytes a thread and
// load), takes max|x| of each as the largest bit pattern (so an infinity or a
// NaN wins), fixes the scales, rescales the page's earlier codes if a scale
// grew, and writes the new codes. Bound by memory, one read and one write of
// the chunk, and by the loads in flight. Measured: 16 prompts of 4096 tokens, 8
// heads of 128, bf16: 69 us for 403 MB, 5.8 TB/s (K and V in CTAs of their own, held
// as fp32: 127); ragged fp32 chunks of 64 sequences, 12 heads of 64: 45 us for
// 195 MB (52), where half of the grid finds no token.

constexpr int KV8_THREADS = 256;

// The larger of every thread's two numbers, each in one word.
__device__ __forceinline__ void block_max2(uint32_t& x, uint32_t& y, uint2* red) {
  x = __reduce_max_sync(0xffffffffu, x);
  y = __reduce_max_sync(0xffffffffu, y);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_uint2(x, y);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KV8_THREADS / 32; ++w) {
    x = max(x, red[w].x);
    y = max(y, red[w].y);
  }
}

// N values (4, 8 or 16) to N codes.
template <int FMT, int N>
__device__ __forceinline__ void kv8_put_codes(uint8_t* p, const float* x, float inv) {
  uint32_t w[N / 4];
#pragma unroll
  for (int u = 0; u < N / 4; ++u) w[u] = kv8_encode4<FMT>(x + 4 * u, inv);
  if constexpr (N == 16)
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (N == 8)
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(p) = w[0];
}

// Scale of a page: what it was, raised to `mine`; NaN if either is.
__device__ __forceinline__ float kv8_raise(float was, float mine) {
  return (was != was || mine != mine) ? __uint_as_float(0x7fc00000u) : fmaxf(was, mine);
}

// Codes of runs [first, last) of a page (held by the threads in turn), and the
// earlier ones rescaled from `was` to `s`.
template <int DT, int FMT, int NG>
__device__ __forceinline__ void kv8_write_page(uint8_t* codes, const uint4 (&x)[NG], int first,
                                               int last, float was, float s) {
  constexpr int N = KV8Type<DT>::N;
  const float inv = kv8_inverse(s);
  // codes of a page whose scale is NaN mean nothing: keep them finite
  const bool spoiled = s != s;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int g = first + threadIdx.x + i * KV8_THREADS;
    if (g < last) {
      float y[N];
      KV8Type<DT>::values(spoiled ? make_uint4(0u, 0u, 0u, 0u) : x[i], y);
      kv8_put_codes<FMT, N>(codes + g * N, y, inv);
    }
  }
  if (first > 0 && !(s == was)) {
    const float ratio = __fmul_rn(was, inv);
    for (int g = threadIdx.x; g < first * (N / 4); g += KV8_THREADS) {
      uint32_t* w = reinterpret_cast<uint32_t*>(codes) + g;
      float y[4];
      kv8_decode4<FMT>(*w, y);
      *w = spoiled ? 0u : kv8_encode4<FMT>(y, ratio);
    }
  }
}

// NG: runs of 16 bytes of K, and of V, that a thread holds.
template <int DT, int NG>
__global__ void __launch_bounds__(KV8_THREADS)
    kv8_append_kernel(KV8 c, const void* __restrict__ k, int64_t k_sb, int64_t k_sh, int64_t k_st,
                      const void* __restrict__ v, int64_t v_sb, int64_t v_sh, int64_t v_st,
                      int vec, const int32_t* __restrict__ counts, int T) {
  constexpr int N = KV8Type<DT>::N;
  __shared__ uint2 red[KV8_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y;
  const int b = blockIdx.z;
  const int len = kv8_len(c, b);
  const int end = kv8_end(c, len, kv8_count(c, counts, b, T));
  const int j = (len >> c.p_shift) + static_cast<int>(blockIdx.x);
  const int p0 = j << c.p_shift;                    // the page's first position
  const int lo = p0 > len ? p0 : len;               // its new tokens are [lo, hi)
  const int hi = p0 + c.P < end ? p0 + c.P : end;
  if (lo >= hi) return;
  const int row_shift = c.d_shift - (N == 8 ? 3 : 2);  // runs of a row, as a power of two
  const int first = (lo - p0) << row_shift, last = (hi - p0) << row_shift;

  // (the loads do not wait for the table)
  uint4 xk[NG], xv[NG];
  const int64_t k0 = b * k_sb + h * k_sh, v0 = b * v_sb + h * v_sh;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int g = first + threadIdx.x + i * KV8_THREADS;
    xk[i] = xv[i] = make_uint4(0u, 0u, 0u, 0u);
    if (g < last) {
      const int r = g >> row_shift, col = N * (g - (r << row_shift));
      const int64_t tok = p0 + r - len;
      xk[i] = KV8Type<DT>::load(k, k0 + tok * k_st + col, vec != 0);
      xv[i] = KV8Type<DT>::load(v, v0 + tok * v_st + col, vec != 0);
    }
  }
  const int page = kv8_page(c, b, j);
  if (page < 0) return;
  const int64_t block = static_cast<int64_t>(page) * c.H + h;
  float2* sp = reinterpret_cast<float2*>(c.scale + 2 * block);
  const float2 was = lo > p0 ? *sp : make_float2(0.f, 0.f);
  uint32_t mk = 0, mv = 0;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    KV8Type<DT>::collect(xk[i], mk);
    KV8Type<DT>::collect(xv[i], mv);
  }
  mk = KV8Type<DT>::bits(mk);
  mv = KV8Type<DT>::bits(mv);
  block_max2(mk, mv, red);
  const float sk = kv8_raise(was.x, kv8_scale(mk, c.fmt));
  const float sv = kv8_raise(was.y, kv8_scale(mv, c.fmt));
  uint8_t* ck = c.k + ((block << c.p_shift) << c.d_shift);
  uint8_t* cv = c.v + ((block << c.p_shift) << c.d_shift);
  if (c.fmt == KF_KV8_INT8) {
    kv8_write_page<DT, KF_KV8_INT8, NG>(ck, xk, first, last, was.x, sk);
    kv8_write_page<DT, KF_KV8_INT8, NG>(cv, xv, first, last, was.y, sv);
  } else {
    kv8_write_page<DT, KF_KV8_E4M3, NG>(ck, xk, first, last, was.x, sk);
    kv8_write_page<DT, KF_KV8_E4M3, NG>(cv, xv, first, last, was.y, sv);
  }
  if (threadIdx.x == 0) *sp = make_float2(sk, sv);
  if (c.weight)
    for (int r = lo - p0 + threadIdx.x; r < hi - p0; r += KV8_THREADS)
      c.weight[block * c.P + r] = 0.f;
}

// ---------------------------------------------------------------- read

// One thread per N codes of K and of V (16 bytes of output each), four rows
// apart in flight. Bound by memory, mostly by what it writes. Measured: 805 MB
// (16 x 8 heads, 8192 tokens of 128, bf16) in 124 us, 6.5 TB/s.
constexpr int KV8_READ_UNROLL = 4;

template <int DT>
__global__ void __launch_bounds__(KV8_THREADS)
    kv8_read_kernel(KV8 c, const int32_t* __restrict__ start, const int32_t* __restrict__ counts,
                    int n, void* __restrict__ k_out, void* __restrict__ v_out) {
  constexpr int N = KV8Type<DT>::N;
  constexpr int W = N / 4;
  pdl_launch_dependents();
  pdl_wait();
  const int row_shift = c.d_shift - (N == 8 ? 3 : 2);
  const int h = blockIdx.y;
  const int b = blockIdx.z;
  const int len = kv8_len(c, b);
  const int end = counts ? kv8_end(c, len, kv8_count(c, counts, b, INT32_MAX)) : len;
  const int from = start ? max(__ldg(start + b), 0) : 0;
  const int64_t out0 = (static_cast<int64_t>(b) * c.H + h) * n * c.D;
  const int total = n << row_shift;
  const int g0 = blockIdx.x * (KV8_THREADS * KV8_READ_UNROLL) + threadIdx.x;
  uint32_t kw[KV8_READ_UNROLL][W], vw[KV8_READ_UNROLL][W];
  float2 s[KV8_READ_UNROLL];
  bool live[KV8_READ_UNROLL];
#pragma unroll
  for (int i = 0; i < KV8_READ_UNROLL; ++i) {
    const int g = g0 + i * KV8_THREADS;
    const int64_t pos = static_cast<int64_t>(from) + (g >> row_shift);
    const bool held = g < total && pos < end;
    bool ok = false;
    const int page = end > 0 ? kv8_page_or0(c, b, held ? static_cast<int>(pos >> c.p_shift) : 0, &ok)
                             : 0;
    if (held && !ok) record_device_status(KF_DEV_BAD_KV_PAGE);
    const int64_t block = static_cast<int64_t>(page) * c.H + h;
    const int64_t at = (((block << c.p_shift) + (pos & (c.P - 1))) << c.d_shift) +
                       N * (g & ((1 << row_shift) - 1));
    s[i] = make_float2(0.f, 0.f);
    if (end > 0) {
      const float2 f = __ldg(reinterpret_cast<const float2*>(c.scale + 2 * block));
      if (held && ok) s[i] = f;
    }
    live[i] = held && ok;
#pragma unroll
    for (int u = 0; u < W; ++u) kw[i][u] = vw[i][u] = 0u;
    if (live[i]) {
      if constexpr (W == 2) {
        const uint2 a = __ldg(reinterpret_cast<const uint2*>(c.k + at));
        const uint2 d = __ldg(reinterpret_cast<const uint2*>(c.v + at));
        kw[i][0] = a.x; kw[i][W - 1] = a.y;
        vw[i][0] = d.x; vw[i][W - 1] = d.y;
      } else {
        kw[i][0] = __ldg(reinterpret_cast<const uint32_t*>(c.k + at));
        vw[i][0] = __ldg(reinterpret_cast<const uint32_t*>(c.v + at));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < KV8_READ_UNROLL; ++i) {
    const int g = g0 + i * KV8_THREADS;
    if (g >= total) return;
    float x[N], y[N];
#pragma unroll
    for (int u = 0; u < W; ++u) {
      if (c.fmt == KF_KV8_INT8) {
        kv8_decode4<KF_KV8_INT8>(kw[i][u], x + 4 * u);
        kv8_decode4<KF_KV8_INT8>(vw[i][u], y + 4 * u);
      } else {
        kv8_decode4<KF_KV8_E4M3>(kw[i][u], x + 4 * u);
        kv8_decode4<KF_KV8_E4M3>(vw[i][u], y + 4 * u);
      }
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      x[u] = __fmul_rn(x[u], s[i].x);
      y[u] = __fmul_rn(y[u], s[i].y);
    }
    const int64_t at = out0 + static_cast<int64_t>(N) * g;
    KV8Type<DT>::store(k_out, at, x);
    KV8Type<DT>::store(v_out, at, y);
  }
}

// ---------------------------------------------------------------- evict
//
// Two kernels. The first picks, per (sequence, kv head), the tokens to keep: a
// radix search, eleven bits a pass, for the need-th largest weight among the
// tokens that are not protected, then a pass in order that lists the kept
// positions. The weights are read from memory once and kept as sortable keys
// in shared memory as far as they fit: a latency chain per row (three searches,
// two passes over its keys). The second moves one destination block per CTA; its
// rows are gathered, 64 to 128 bytes each. Measured, 16 x 8 heads of 24k tokens
// cut to 8192 of 128: selection 36 us, move 127 us for 537 MB (4.2 TB/s).

constexpr int KV8_SELECT_THREADS = 1024;
constexpr int KV8_SELECT_KEYS = 48 * 1024;  // keys that shared memory holds
constexpr int KV8_SELECT_SMEM = KV8_SELECT_KEYS * 4;

// Weights in an order of unsigned integers; NaN counts as the largest, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(__fadd_rn(w, 0.f));
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(KV8_SELECT_THREADS)
    kv8_select_kernel(KV8 c, int budget, int recent, int32_t* __restrict__ kept,
                      int32_t* __restrict__ lens_out) {
  extern __shared__ uint32_t s_key[];  // [KV8_SELECT_KEYS]
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t s_part[32];
  __shared__ uint32_t s_prefix, s_need;
  __shared__ uint32_t w_more[32], w_tie[32];
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.x;
  const int b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = kv8_len(c, b);
  const int n = len < budget ? len : budget;
  int32_t* out = kept + (static_cast<int64_t>(b) * c.H + h) * budget;
  if (h == 0 && tid == 0) lens_out[b] = n;
  if (len <= budget) {
    for (int i = tid; i < budget; i += KV8_SELECT_THREADS) out[i] = i < len ? i : -1;
    return;
  }
  const int cand = len - recent;           // positions [0, cand) compete
  const int need = budget - recent;        // for this many places (need < cand)
  for (int i = tid; i < recent; i += KV8_SELECT_THREADS) out[need + i] = cand + i;
  if (need == 0) return;
  auto load_key = [&](int pos) -> uint32_t {
    bool ok;
    const int page = kv8_page_or0(c, b, pos >> c.p_shift, &ok);
    const float x = c.weight[(static_cast<int64_t>(page) * c.H + h) * c.P + (pos & (c.P - 1))];
    return ok ? weight_key(x) : 0u;
  };
  // Eight keys a thread at a time: all table entries, then all weights (a
  // refused page is recorded after them, or its branch would order the loads).
  bool bad = false;
  for (int base = tid; base < cand; base += 8 * KV8_SELECT_THREADS) {
    int page[8];
    float x[8];
    bool ok[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pos = base + i * KV8_SELECT_THREADS;
      page[i] = kv8_page_or0(c, b, (pos < cand ? pos : 0) >> c.p_shift, &ok[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pos = base + i * KV8_SELECT_THREADS;
      x[i] = c.weight[(static_cast<int64_t>(page[i]) * c.H + h) * c.P + (pos & (c.P - 1))];
      bad = bad || !ok[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pos = base + i * KV8_SELECT_THREADS;
      if (pos < cand && pos < KV8_SELECT_KEYS) s_key[pos] = ok[i] ? weight_key(x[i]) : 0u;
    }
  }
  if (bad) record_device_status(KF_DEV_BAD_KV_PAGE);
  auto key_at = [&](int pos) -> uint32_t {
    return pos < KV8_SELECT_KEYS ? s_key[pos] : load_key(pos);
  };
  // The need-th largest key, eleven bits at a time: s_prefix holds the bits
  // found, s_need how many keys with that prefix still have to be taken.
  if (tid == 0) {
    s_prefix = 0;
    s_need = need;
  }
  int left_bits = 32;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10;
    const int shift = left_bits - bits;
    const uint32_t above = pass == 0 ? 0u : (0xffffffffu << left_bits);
    hist[tid] = 0;
    hist[tid + 1024] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix, want = s_need;
    for (int pos = tid; pos < cand; pos += KV8_SELECT_THREADS) {
      const uint32_t key = key_at(pos);
      if ((key & above) == prefix) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1u)], 1u);
    }
    __syncthreads();
    // Thread i looks at digits 2047 - 2i and 2046 - 2i: a scan over the threads
    // counts the keys with larger digits; one thread finds its digit is it.
    const uint32_t h0 = hist[2047 - 2 * tid], h1 = hist[2046 - 2 * tid];
    uint32_t sum = h0 + h1;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) s_part[warp] = sum;
    __syncthreads();
    uint32_t before = sum - h0 - h1;
    for (int w = 0; w < warp; ++w) before += s_part[w];
    if (before < want && before + h0 >= want) {
      s_prefix = prefix | (static_cast<uint32_t>(2047 - 2 * tid) << shift);
      s_need = want - before;
    } else if (before + h0 < want && before + h0 + h1 >= want) {
      s_prefix = prefix | (static_cast<uint32_t>(2046 - 2 * tid) << shift);
      s_need = want - before - h0;
    }
    left_bits = shift;
    __syncthreads();
  }
  const uint32_t cut = s_prefix;
  const uint32_t ties = s_need;  // keys equal to cut that are kept, lowest position first
  // Every warp takes a run of positions: it counts, then lists, what it keeps.
  const int run = ((cand + 31) / 32 + 31) / 32 * 32;
  const int begin = warp * run, stop = min(begin + run, cand);
  uint32_t more = 0, tie = 0;
  for (int pos = begin + lane; pos < begin + run; pos += 32) {
    const uint32_t key = pos < stop ? key_at(pos) : 0u;
    more += __popc(__ballot_sync(0xffffffffu, pos < stop && key > cut));
    tie += __popc(__ballot_sync(0xffffffffu, pos < stop && key == cut));
  }
  if (lane == 0) {
    w_more[warp] = more;
    w_tie[warp] = tie;
  }
  __syncthreads();
  uint32_t pm = 0, pt = 0;
  for (int w = 0; w < warp; ++w) {
    pm += w_more[w];
    pt += w_tie[w];
  }
  const uint32_t below = (1u << lane) - 1u;
  for (int pos = begin + lane; pos < begin + run; pos += 32) {
    const uint32_t key = pos < stop ? key_at(pos) : 0u;
    const bool is_more = pos < stop && key > cut, is_tie = pos < stop && key == cut;
    const uint32_t bm = __ballot_sync(0xffffffffu, is_more);
    const uint32_t bt = __ballot_sync(0xffffffffu, is_tie);
    const uint32_t m = pm + __popc(bm & below), t = pt + __popc(bt & below);
    if (is_more || (is_tie && t < ties)) out[m + min(t, ties)] = pos;
    pm += __popc(bm);
    pt += __popc(bt);
  }
}

// Largest |code| of 16 codes, as fp16 (exact).
template <int FMT>
__device__ __forceinline__ float kv8_top16(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  __half2 m = __half2half2(__ushort_as_half(0));
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    uint32_t a, b;
    kv8_cvt4<FMT>(w[u], a, b);
    m = __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&a)));
    m = __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&b)));
  }
  return fmaxf(__low2float(m), __high2float(m));
}

// The values of 16 codes under scale s, quantised with 1 / scale `inv`.
template <int FMT>
__device__ __forceinline__ void kv8_recode16(uint8_t* p, const uint4& v, float s, float inv) {
  float x[16];
  kv8_decode4<FMT>(v.x, x);
  kv8_decode4<FMT>(v.y, x + 4);
  kv8_decode4<FMT>(v.z, x + 8);
  kv8_decode4<FMT>(v.w, x + 12);
#pragma unroll
  for (int u = 0; u < 16; ++u) x[u] = __fmul_rn(x[u], s);
  kv8_put_codes<FMT, 16>(p, x, inv);
}

// NG: pieces of 16 codes of K, and of V, that a thread moves. A row's scale is
// the same along it, so the largest value of a piece is its largest code
// times that (rounding keeps the order): the codes are decoded once.
template <int FMT, int NG>
__global__ void __launch_bounds__(KV8_THREADS, NG <= 2 ? 5 : 3)
    kv8_move_kernel(KV8 c, const int32_t* __restrict__ table_out, int64_t ld_out, int budget,
                    const int32_t* __restrict__ kept) {
  __shared__ uint2 red[KV8_THREADS / 32];
  __shared__ int64_t s_row[128];     // source row (block * P + slot) of each destination slot
  __shared__ float2 s_scale[128];
  pdl_launch_dependents();
  pdl_wait();
  const int j = blockIdx.x;
  const int h = blockIdx.y;
  const int b = blockIdx.z;
  const int len = kv8_len(c, b);
  const int n = len < budget ? len : budget;
  const int p0 = j << c.p_shift;
  const int rows = n - p0 < c.P ? n - p0 : c.P;
  if (rows <= 0) return;
  const int page = kv8_page(c, table_out, ld_out, b, j);
  if (page < 0) return;
  const int64_t block = static_cast<int64_t>(page) * c.H + h;
  const int32_t* mine = kept + (static_cast<int64_t>(b) * c.H + h) * budget + p0;
  if (threadIdx.x < rows) {
    const int pos = mine[threadIdx.x];
    const int sp = kv8_page(c, b, pos >> c.p_shift);
    const int64_t from = static_cast<int64_t>(sp) * c.H + h;
    const int64_t row = sp < 0 ? -1 : from * c.P + (pos & (c.P - 1));
    s_row[threadIdx.x] = row;
    s_scale[threadIdx.x] =
        sp < 0 ? make_float2(0.f, 0.f) : *reinterpret_cast<const float2*>(c.scale + 2 * from);
    c.weight[block * c.P + threadIdx.x] = row >= 0 ? c.weight[row] : 0.f;
  }
  __syncthreads();
  const int row_shift = c.d_shift - 4;
  const int last = rows << row_shift;
  uint4 wk[NG], wv[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int g = threadIdx.x + i * KV8_THREADS;
    wk[i] = wv[i] = make_uint4(0u, 0u, 0u, 0u);
    if (g < last) {
      const int64_t row = s_row[g >> row_shift];
      const int64_t at = (row << c.d_shift) + 16 * (g & ((1 << row_shift) - 1));
      if (row >= 0) {
        wk[i] = *reinterpret_cast<const uint4*>(c.k + at);
        wv[i] = *reinterpret_cast<const uint4*>(c.v + at);
      }
    }
  }
  uint32_t mk = 0, mv = 0;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int g = threadIdx.x + i * KV8_THREADS;
    const float2 s = g < last ? s_scale[g >> row_shift] : make_float2(0.f, 0.f);
    mk = max(mk, __float_as_uint(__fmul_rn(kv8_top16<FMT>(wk[i]), s.x)) & 0x7fffffffu);
    mv = max(mv, __float_as_uint(__fmul_rn(kv8_top16<FMT>(wv[i]), s.y)) & 0x7fffffffu);
  }
  block_max2(mk, mv, red);
  const float sk = kv8_scale(mk, c.fmt), sv = kv8_scale(mv, c.fmt);
  const float ik = kv8_inverse(sk), iv = kv8_inverse(sv);
  const int64_t base = (block << c.p_shift) << c.d_shift;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int g = threadIdx.x + i * KV8_THREADS;
    if (g < last) {
      const float2 s = s_scale[g >> row_shift];
      // (a NaN scale makes the block's NaN: its codes are 0)
      kv8_recode16<FMT>(c.k + base + 16 * g, wk[i], sk == sk ? s.x : 0.f, ik);
      kv8_recode16<FMT>(c.v + base + 16 * g, wv[i], sv == sv ? s.y : 0.f, iv);
    }
  }
  if (threadIdx.x == 0) *reinterpret_cast<float2*>(c.scale + 2 * block) = make_float2(sk, sv);
}

// ---------------------------------------------------------------- host

static int log2_exact(int x) {
  for (int s = 0; s < 31; ++s)
    if (x == (1 << s)) return s;
  return -1;
}

// Checks a cache description; fills the device view.
static int kv8_view(const char* what, const kf_kv8_cache* c, KV8* out) {
  // (tensors without elements have no address)
  if (!c || (c->pages && (!c->k || !c->v || !c->scale)) ||
      (c->batch && ((c->blocks && !c->table) || !c->lens)) || c->pages < 0 || c->batch < 0 ||
      c->kv_heads <= 0 || c->blocks < 0 || c->ld_table < c->blocks) {
    set_last_error("%s: invalid cache (null pointer, negative size or ld_table < blocks)", what);
    return KF_E_INVALID;
  }
  if (c->format != KF_KV8_INT8 && c->format != KF_KV8_E4M3) {
    set_last_error("%s: unknown code format %d", what, c->format);
    return KF_E_INVALID;
  }
  if (c->head_dim != 16 && c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) {
    set_last_error("%s: head_dim %d not in {16, 32, 64, 128}", what, c->head_dim);
    return KF_E_UNSUPPORTED;
  }
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) {
    set_last_error("%s: block %d not in {16, 32, 64, 128}", what, c->block);
    return KF_E_UNSUPPORTED;
  }
  if (!kv8_aligned(c->k, 16) || !kv8_aligned(c->v, 16) || !kv8_aligned(c->scale, 8)) {
    set_last_error("%s: codes must be 16-byte and scales 8-byte aligned", what);
    return KF_E_UNSUPPORTED;
  }
  if (c->batch > 32767 || c->kv_heads > 65535 || c->pages > INT32_MAX ||
      static_cast<int64_t>(c->blocks) * c->block > INT32_MAX / 2) {
    set_last_error("%s: needs batch <= 32767, kv_heads <= 65535, pages < 2^31 and a table that "
                   "reaches fewer than 2^30 tokens", what);
    return KF_E_UNSUPPORTED;
  }
  KV8 v;
  v.k = static_cast<uint8_t*>(c->k);
  v.v = static_cast<uint8_t*>(c->v);
  v.scale = c->scale;
  v.weight = c->weight;
  v.table = c->table;
  v.lens = c->lens;
  v.pages = c->pages;
  v.ld_table = c->ld_table;
  v.blocks = c->pages ? c->blocks : 0;  // an empty pool holds no token
  v.B = c->batch;
  v.H = c->kv_heads;
  v.D = c->head_dim;
  v.P = c->block;
  v.fmt = c->format;
  v.p_shift = log2_exact(c->block);
  v.d_shift = log2_exact(c->head_dim);
  *out = v;
  return KF_OK;
}

static int kv8_dtype(const char* what, int dtype) {
  if (dtype == KF_DT_F32 || dtype == KF_DT_BF16 || dtype == KF_DT_F16) return KF_OK;
  set_last_error("%s: unknown element type %d", what, dtype);
  return KF_E_INVALID;
}
static int64_t dtype_size(int dtype) { return dtype == KF_DT_F32 ? 4 : 2; }

}  // namespace kf

using namespace kf;

extern "C" int kf_kv8_append(const kf_kv8_cache* cache, const void* k, int64_t k_sb, int64_t k_sh,
                             int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st,
                             int dtype, const int32_t* counts, int64_t T, void* stream) {
  KV8 c;
  int rc = kv8_view("kf_kv8_append", cache, &c);
  if (!rc) rc = kv8_dtype("kf_kv8_append", dtype);
  if (rc) return rc;
  if (T == 0 || c.B == 0) return KF_OK;
  if (!k || !v || T < 0 || T > INT32_MAX / 2) {
    set_last_error("kf_kv8_append: invalid arguments (T = %lld)", (long long)T);
    return KF_E_INVALID;
  }
  const int64_t es = dtype_size(dtype), per = 16 / es;
  const int64_t strides[6] = {k_sb, k_sh, k_st, v_sb, v_sh, v_st};
  int vec = kv8_aligned(k, 16) && kv8_aligned(v, 16);
  for (int i = 0; i < 6; ++i) vec = vec && strides[i] % per == 0;
  const unsigned n = static_cast<unsigned>((c.P + T - 2) / c.P + 1);
  const dim3 grid(n, static_cast<unsigned>(c.H), static_cast<unsigned>(c.B));
  // runs of 16 bytes that a thread holds: of a page, or of a chunk that is shorter
  const int64_t rows = T < c.P ? T : c.P;
  const int64_t groups = (rows * c.D / per + KV8_THREADS - 1) / KV8_THREADS;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int Ti = static_cast<int>(T);
  cudaError_t e;
#define KF_KV8_APPEND(DT, NG)                                                                    \
  e = launch_chained(kv8_append_kernel<DT, NG>, grid, dim3(KV8_THREADS), 0, st, c, k, k_sb, k_sh, \
                     k_st, v, v_sb, v_sh, v_st, vec, counts, Ti)
#define KF_KV8_APPEND_NG(DT)      \
  do {                            \
    if (groups <= 1)              \
      KF_KV8_APPEND(DT, 1);       \
    else if (groups <= 2)         \
      KF_KV8_APPEND(DT, 2);       \
    else if (groups <= 4)         \
      KF_KV8_APPEND(DT, 4);       \
    else                          \
      KF_KV8_APPEND(DT, 8);       \
  } while (0)
  if (dtype == KF_DT_F32 && groups > 8)  // a whole page of 128 x 128
    KF_KV8_APPEND(KF_DT_F32, 16);
  else if (dtype == KF_DT_F32)
    KF_KV8_APPEND_NG(KF_DT_F32);
  else if (dtype == KF_DT_BF16)
    KF_KV8_APPEND_NG(KF_DT_BF16);
  else
    KF_KV8_APPEND_NG(KF_DT_F16);
#undef KF_KV8_APPEND_NG
#undef KF_KV8_APPEND
  return cuda_status(e, "kf_kv8_append launch");
}

extern "C" int kf_kv8_read(const kf_kv8_cache* cache, const int32_t* start, const int32_t* counts,
                           int64_t n, void* k_out, void* v_out, int dtype, void* stream) {
  KV8 c;
  int rc = kv8_view("kf_kv8_read", cache, &c);
  if (!rc) rc = kv8_dtype("kf_kv8_read", dtype);
  if (rc) return rc;
  if (n == 0 || c.B == 0) return KF_OK;
  if (!k_out || !v_out || n < 0 || n > INT32_MAX / c.D) {
    set_last_error("kf_kv8_read: invalid arguments (n = %lld)", (long long)n);
    return KF_E_INVALID;
  }
  if (!kv8_aligned(k_out, 16) || !kv8_aligned(v_out, 16)) {
    set_last_error("kf_kv8_read: outputs must be 16-byte aligned");
    return KF_E_UNSUPPORTED;
  }
  const int64_t groups = n * c.D * dtype_size(dtype) / 16;
  constexpr int64_t per_cta = KV8_THREADS * KV8_READ_UNROLL;
  const dim3 grid(static_cast<unsigned>((groups + per_cta - 1) / per_cta),
                  static_cast<unsigned>(c.H), static_cast<unsigned>(c.B));
  auto kern = dtype == KF_DT_F32    ? kv8_read_kernel<KF_DT_F32>
              : dtype == KF_DT_BF16 ? kv8_read_kernel<KF_DT_BF16>
                                    : kv8_read_kernel<KF_DT_F16>;
  return cuda_status(launch_chained(kern, grid, dim3(KV8_THREADS), 0,
                                    static_cast<cudaStream_t>(stream), c, start, counts,
                                    static_cast<int>(n), k_out, v_out),
                     "kf_kv8_read launch");
}

extern "C" int kf_kv8_evict(const kf_kv8_cache* cache, const int32_t* table_out, int64_t ld_out,
                            int64_t budget, int64_t recent, int32_t* kept, int32_t* lens_out,
                            void* stream) {
  KV8 c;
  int rc = kv8_view("kf_kv8_evict", cache, &c);
  if (rc) return rc;
  if ((c.B && (!table_out || !kept || !lens_out)) || budget <= 0 || recent < 0 || recent > budget ||
      budget > INT32_MAX / 2 || ld_out * c.P < budget) {
    set_last_error("kf_kv8_evict: needs 0 <= recent <= budget, budget > 0 and a table_out that "
                   "holds budget tokens (budget %lld, recent %lld)",
                   (long long)budget, (long long)recent);
    return KF_E_INVALID;
  }
  if (c.B && lens_out == c.lens) {
    set_last_error("kf_kv8_evict: lens_out must not be the cache's lens");
    return KF_E_INVALID;
  }
  if (c.pages && !c.weight) {
    set_last_error("kf_kv8_evict: the cache keeps no weight record");
    return KF_E_INVALID;
  }
  if (c.B == 0) return KF_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int bud = static_cast<int>(budget), rec = static_cast<int>(recent);
  static DeviceOnce once;
  rc = once.run("kf_kv8_evict", nullptr, [&](int) {
    return cuda_status(cudaFuncSetAttribute(kv8_select_kernel,
                                            cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            KV8_SELECT_SMEM),
                       "kf_kv8_evict: set smem attribute");
  });
  if (rc) return rc;
  // no more keys in shared memory than a table can hold
  const int64_t reach = static_cast<int64_t>(c.blocks) * c.P;
  const size_t smem = reach < KV8_SELECT_KEYS ? static_cast<size_t>(reach) * 4 : KV8_SELECT_SMEM;
  cudaError_t e = launch_chained(kv8_select_kernel,
                                 dim3(static_cast<unsigned>(c.H), static_cast<unsigned>(c.B)),
                                 dim3(KV8_SELECT_THREADS), smem, st, c, bud, rec, kept, lens_out);
  if (e != cudaSuccess) return cuda_status(e, "kf_kv8_evict select launch");
  const dim3 grid(static_cast<unsigned>((budget + c.P - 1) / c.P), static_cast<unsigned>(c.H),
                  static_cast<unsigned>(c.B));
  const int groups = c.P * c.D / 16 / KV8_THREADS;
#define KF_KV8_MOVE(FMT, NG)                                                                    \
  e = launch_chained(kv8_move_kernel<FMT, NG>, grid, dim3(KV8_THREADS), 0, st, c, table_out,     \
                     ld_out, bud, static_cast<const int32_t*>(kept))
#define KF_KV8_MOVE_NG(FMT)    \
  do {                         \
    if (groups <= 1)           \
      KF_KV8_MOVE(FMT, 1);     \
    else if (groups <= 2)      \
      KF_KV8_MOVE(FMT, 2);     \
    else                       \
      KF_KV8_MOVE(FMT, 4);     \
  } while (0)
  if (c.fmt == KF_KV8_INT8)
    KF_KV8_MOVE_NG(KF_KV8_INT8);
  else
    KF_KV8_MOVE_NG(KF_KV8_E4M3);
#undef KF_KV8_MOVE_NG
#undef KF_KV8_MOVE
  return cuda_status(e, "kf_kv8_evict move launch");
}
