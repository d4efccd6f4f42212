// Writing, reading and thinning the 8-bit key/value cache.
#include "kv8_common.cuh"

namespace kf {

// ---------------------------------------------------------------- append
//
// One CTA per (page a chunk can reach, kv head, sequence and K|V). It loads the
// page's new tokens into registers, takes max|x| as the largest bit pattern
// (so an infinity or a NaN wins), fixes the scale, rescales the page's earlier
// codes if the scale grew, and writes the new codes.

constexpr int KV8_THREADS = 256;

__device__ __forceinline__ uint32_t block_max_u32(uint32_t x, uint32_t* red) {
  x = __reduce_max_sync(0xffffffffu, x);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  uint32_t m = red[0];
#pragma unroll
  for (int w = 1; w < KV8_THREADS / 32; ++w) m = max(m, red[w]);
  return m;
}

// 4 values to 4 codes, one word.
__device__ __forceinline__ uint32_t kv8_encode4(const float (&x)[4], float inv, int fmt) {
  uint32_t w = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    w |= static_cast<uint32_t>(kv8_encode(__fmul_rn(x[u], inv), fmt)) << (8 * u);
  return w;
}
__device__ __forceinline__ void kv8_decode4(uint32_t w, int fmt, float (&x)[4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) x[u] = kv8_decode(static_cast<uint8_t>(w >> (8 * u)), fmt);
}

// NG: groups of four values a thread holds (a page has P * D / 4 groups).
template <int NG>
__global__ void __launch_bounds__(KV8_THREADS)
    kv8_append_kernel(KV8 c, const void* __restrict__ k, int64_t k_sb, int64_t k_sh, int64_t k_st,
                      const void* __restrict__ v, int64_t v_sb, int64_t v_sh, int64_t v_st,
                      int dtype, int vec, const int32_t* __restrict__ counts, int T) {
  __shared__ uint32_t red[KV8_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y;
  const int b = blockIdx.z >> 1;
  const bool is_v = blockIdx.z & 1;
  const int len = kv8_len(c, b);
  const int end = kv8_end(c, len, kv8_count(counts, b, T));
  const int j = (len >> c.p_shift) + static_cast<int>(blockIdx.x);
  const int p0 = j << c.p_shift;                    // the page's first position
  const int lo = p0 > len ? p0 : len;               // its new tokens are [lo, hi)
  const int hi = p0 + c.P < end ? p0 + c.P : end;
  if (lo >= hi) return;
  const int page = kv8_page(c, b, j);
  if (page < 0) return;

  const void* src = is_v ? v : k;
  const int64_t base = b * (is_v ? v_sb : k_sb) + h * (is_v ? v_sh : k_sh);
  const int64_t st = is_v ? v_st : k_st;
  const int64_t block = static_cast<int64_t>(page) * c.H + h;
  uint32_t* codes = reinterpret_cast<uint32_t*>((is_v ? c.v : c.k) + block * c.P * c.D);
  float* sp = c.scale + 2 * block + (is_v ? 1 : 0);
  const float was = lo > p0 ? *sp : 0.f;
  const int row_groups = c.D >> 2;
  const int first = (lo - p0) * row_groups, last = (hi - p0) * row_groups;

  float x[NG][4];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int g = first + threadIdx.x + i * KV8_THREADS;
    x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
    if (g < last) {
      const int r = g / row_groups;
      kv8_load4(src, base + (p0 + r - len) * st + 4 * (g - r * row_groups), dtype, vec, x[i]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) amax = max(amax, __float_as_uint(x[i][u]) & 0x7fffffffu);
  }
  const float mine = kv8_scale(block_max_u32(amax, red), c.fmt);
  const float s = (was != was || mine != mine) ? __uint_as_float(0x7fc00000u) : fmaxf(was, mine);
  const float inv = kv8_inverse(s);
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int g = first + threadIdx.x + i * KV8_THREADS;
    if (g < last) codes[g] = kv8_encode4(x[i], inv, c.fmt);
  }
  if (first > 0 && !(s == was)) {
    const float ratio = __fmul_rn(was, inv);
    for (int g = threadIdx.x; g < first; g += KV8_THREADS) {
      float y[4];
      kv8_decode4(codes[g], c.fmt, y);
      codes[g] = kv8_encode4(y, ratio, c.fmt);
    }
  }
  if (threadIdx.x == 0) *sp = s;
  if (c.weight && !is_v)
    for (int r = lo - p0 + threadIdx.x; r < hi - p0; r += KV8_THREADS)
      c.weight[block * c.P + r] = 0.f;
}

// ---------------------------------------------------------------- read

// One thread per four codes of K or V.
__global__ void __launch_bounds__(KV8_THREADS)
    kv8_read_kernel(KV8 c, const int32_t* __restrict__ start, const int32_t* __restrict__ counts,
                    int n, void* __restrict__ k_out, void* __restrict__ v_out, int dtype) {
  pdl_launch_dependents();
  pdl_wait();
  const int row_groups = c.D >> 2;
  const int h = blockIdx.y;
  const int b = blockIdx.z;
  const int len = kv8_len(c, b);
  const int end = counts ? kv8_end(c, len, max(__ldg(counts + b), 0)) : len;
  const int from = start ? max(__ldg(start + b), 0) : 0;
  const int64_t out0 = (static_cast<int64_t>(b) * c.H + h) * n * c.D;
  const int total = n * row_groups;
  for (int g = blockIdx.x * KV8_THREADS + threadIdx.x; g < total; g += gridDim.x * KV8_THREADS) {
    const int i = g / row_groups;
    const int64_t pos = static_cast<int64_t>(from) + i;
    float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
    if (pos < end) {
      const int page = kv8_page(c, b, static_cast<int>(pos >> c.p_shift));
      if (page >= 0) {
        const int64_t block = static_cast<int64_t>(page) * c.H + h;
        const int64_t at = (block * c.P + (pos & (c.P - 1))) * row_groups + (g - i * row_groups);
        const float2 s = *reinterpret_cast<const float2*>(c.scale + 2 * block);
        kv8_decode4(reinterpret_cast<const uint32_t*>(c.k)[at], c.fmt, x);
        kv8_decode4(reinterpret_cast<const uint32_t*>(c.v)[at], c.fmt, y);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          x[u] = __fmul_rn(x[u], s.x);
          y[u] = __fmul_rn(y[u], s.y);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      kv8_store1(k_out, out0 + 4 * static_cast<int64_t>(g) + u, dtype, x[u]);
      kv8_store1(v_out, out0 + 4 * static_cast<int64_t>(g) + u, dtype, y[u]);
    }
  }
}

// ---------------------------------------------------------------- evict
//
// Two kernels. The first picks, per (sequence, kv head), the tokens to keep:
// a radix search, eight bits a pass, for the need-th largest weight among the
// tokens that are not protected, then one pass in order that lists the kept
// positions. The second moves one destination block per CTA.

constexpr int KV8_SELECT_THREADS = 1024;

// Weights in an order of unsigned integers; NaN counts as the largest, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(__fadd_rn(w, 0.f));
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(KV8_SELECT_THREADS)
    kv8_select_kernel(KV8 c, int budget, int recent, int32_t* __restrict__ kept,
                      int32_t* __restrict__ lens_out) {
  __shared__ uint32_t hist[256];
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
  auto key_at = [&](int pos) -> uint32_t {
    const int page = kv8_page(c, b, pos >> c.p_shift);
    if (page < 0) return 0u;
    return weight_key(
        c.weight[(static_cast<int64_t>(page) * c.H + h) * c.P + (pos & (c.P - 1))]);
  };
  // The need-th largest key, eight bits at a time: s_prefix holds the bits
  // found, s_need how many keys with that prefix still have to be taken.
  if (tid == 0) {
    s_prefix = 0;
    s_need = need;
  }
  for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix;
    const uint32_t above = shift == 24 ? 0u : (0xffffffffu << (shift + 8));
    for (int pos = tid; pos < cand; pos += KV8_SELECT_THREADS) {
      const uint32_t key = key_at(pos);
      if ((key & above) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t left = s_need;
      int d = 255;
      while (d > 0 && hist[d] < left) left -= hist[d--];
      s_prefix = prefix | (static_cast<uint32_t>(d) << shift);
      s_need = left;
    }
    __syncthreads();
  }
  __syncthreads();
  const uint32_t cut = s_prefix;
  const uint32_t ties = need > 0 ? s_need : 0u;  // keys equal to cut that are kept, lowest first
  uint32_t more_before = 0, tie_before = 0;
  for (int base = 0; base < cand && need > 0; base += KV8_SELECT_THREADS) {
    const int pos = base + tid;
    const uint32_t key = pos < cand ? key_at(pos) : 0u;
    const bool more = pos < cand && key > cut;
    const bool tie = pos < cand && key == cut;
    const uint32_t bm = __ballot_sync(0xffffffffu, more), bt = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) {
      w_more[warp] = __popc(bm);
      w_tie[warp] = __popc(bt);
    }
    __syncthreads();
    uint32_t pm = more_before, pt = tie_before, all_m = 0, all_t = 0;
    for (int w = 0; w < 32; ++w) {
      if (w == warp) {
        pm += all_m;
        pt += all_t;
      }
      all_m += w_more[w];
      all_t += w_tie[w];
    }
    const uint32_t below = (1u << lane) - 1u;
    pm += __popc(bm & below);
    pt += __popc(bt & below);
    if (more || (tie && pt < ties)) out[pm + (pt < ties ? pt : ties)] = pos;
    more_before += all_m;
    tie_before += all_t;
    __syncthreads();
  }
  for (int i = tid; i < recent; i += KV8_SELECT_THREADS) out[need + i] = cand + i;
}

template <int NG>
__global__ void __launch_bounds__(KV8_THREADS)
    kv8_move_kernel(KV8 c, const int32_t* __restrict__ table_out, int64_t ld_out, int budget,
                    const int32_t* __restrict__ kept) {
  __shared__ uint32_t red[KV8_THREADS / 32];
  __shared__ int64_t s_row[128];     // source row (block * P + slot) of each destination slot
  pdl_launch_dependents();
  pdl_wait();
  const int j = blockIdx.x;
  const int h = blockIdx.y;
  const int b = blockIdx.z >> 1;
  const bool is_v = blockIdx.z & 1;
  const int len = kv8_len(c, b);
  const int n = len < budget ? len : budget;
  const int p0 = j << c.p_shift;
  const int rows = n - p0 < c.P ? n - p0 : c.P;
  if (rows <= 0) return;
  const int page = kv8_page(c, table_out, ld_out, b, j);
  if (page < 0) return;
  const int32_t* mine = kept + (static_cast<int64_t>(b) * c.H + h) * budget + p0;
  if (threadIdx.x < rows) {
    const int pos = mine[threadIdx.x];
    const int sp = kv8_page(c, b, pos >> c.p_shift);
    s_row[threadIdx.x] =
        sp < 0 ? -1 : (static_cast<int64_t>(sp) * c.H + h) * c.P + (pos & (c.P - 1));
  }
  __syncthreads();
  const int row_groups = c.D >> 2;
  const uint32_t* src = reinterpret_cast<const uint32_t*>(is_v ? c.v : c.k);
  const int last = rows * row_groups;
  float x[NG][4];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int g = threadIdx.x + i * KV8_THREADS;
    x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
    if (g < last) {
      const int r = g / row_groups;
      const int64_t row = s_row[r];
      if (row >= 0) {
        const float s = c.scale[2 * (row >> c.p_shift) + (is_v ? 1 : 0)];
        kv8_decode4(src[row * row_groups + (g - r * row_groups)], c.fmt, x[i]);
#pragma unroll
        for (int u = 0; u < 4; ++u) x[i][u] = __fmul_rn(x[i][u], s);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) amax = max(amax, __float_as_uint(x[i][u]) & 0x7fffffffu);
  }
  const float s = kv8_scale(block_max_u32(amax, red), c.fmt);
  const float inv = kv8_inverse(s);
  const int64_t block = static_cast<int64_t>(page) * c.H + h;
  uint32_t* codes = reinterpret_cast<uint32_t*>((is_v ? c.v : c.k) + block * c.P * c.D);
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int g = threadIdx.x + i * KV8_THREADS;
    if (g < last) codes[g] = kv8_encode4(x[i], inv, c.fmt);
  }
  if (threadIdx.x == 0) c.scale[2 * block + (is_v ? 1 : 0)] = s;
  if (!is_v && threadIdx.x < rows) {
    const int64_t row = s_row[threadIdx.x];
    c.weight[block * c.P + threadIdx.x] = row >= 0 ? c.weight[row] : 0.f;
  }
}

// ---------------------------------------------------------------- host

static int log2_exact(int x) {
  for (int s = 0; s < 31; ++s)
    if (x == (1 << s)) return s;
  return -1;
}

// Checks a cache description; fills the device view.
static int kv8_view(const char* what, const kf_kv8_cache* c, KV8* out) {
  if (!c || !c->k || !c->v || !c->scale || !c->table || !c->lens || c->pages < 0 ||
      c->batch < 0 || c->kv_heads <= 0 || c->blocks < 0 || c->ld_table < c->blocks) {
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
  const int64_t es = dtype_size(dtype);
  const int64_t strides[6] = {k_sb, k_sh, k_st, v_sb, v_sh, v_st};
  int vec = kv8_aligned(k, 4 * es) && kv8_aligned(v, 4 * es);
  for (int i = 0; i < 6; ++i) vec = vec && strides[i] % 4 == 0;
  const unsigned n = static_cast<unsigned>((c.P + T - 2) / c.P + 1);
  const dim3 grid(n, static_cast<unsigned>(c.H), static_cast<unsigned>(2 * c.B));
  const int groups = c.P * c.D / 4 / KV8_THREADS;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int Ti = static_cast<int>(T);
  cudaError_t e;
#define KF_KV8_APPEND(NG)                                                                        \
  e = launch_chained(kv8_append_kernel<NG>, grid, dim3(KV8_THREADS), 0, st, c, k, k_sb, k_sh,    \
                     k_st, v, v_sb, v_sh, v_st, dtype, vec, counts, Ti)
  if (groups <= 1)
    KF_KV8_APPEND(1);
  else if (groups <= 2)
    KF_KV8_APPEND(2);
  else if (groups <= 4)
    KF_KV8_APPEND(4);
  else if (groups <= 8)
    KF_KV8_APPEND(8);
  else
    KF_KV8_APPEND(16);
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
  const int64_t groups = n * c.D / 4;
  const dim3 grid(static_cast<unsigned>((groups + KV8_THREADS - 1) / KV8_THREADS),
                  static_cast<unsigned>(c.H), static_cast<unsigned>(c.B));
  return cuda_status(launch_chained(kv8_read_kernel, grid, dim3(KV8_THREADS), 0,
                                    static_cast<cudaStream_t>(stream), c, start, counts,
                                    static_cast<int>(n), k_out, v_out, dtype),
                     "kf_kv8_read launch");
}

extern "C" int kf_kv8_evict(const kf_kv8_cache* cache, const int32_t* table_out, int64_t ld_out,
                            int64_t budget, int64_t recent, int32_t* kept, int32_t* lens_out,
                            void* stream) {
  KV8 c;
  int rc = kv8_view("kf_kv8_evict", cache, &c);
  if (rc) return rc;
  if (!table_out || !kept || !lens_out || budget <= 0 || recent < 0 || recent > budget ||
      budget > INT32_MAX / 2 || ld_out * c.P < budget) {
    set_last_error("kf_kv8_evict: needs 0 <= recent <= budget, budget > 0 and a table_out that "
                   "holds budget tokens (budget %lld, recent %lld)",
                   (long long)budget, (long long)recent);
    return KF_E_INVALID;
  }
  if (lens_out == c.lens) {
    set_last_error("kf_kv8_evict: lens_out must not be the cache's lens");
    return KF_E_INVALID;
  }
  if (!c.weight) {
    set_last_error("kf_kv8_evict: the cache keeps no weight record");
    return KF_E_INVALID;
  }
  if (c.B == 0) return KF_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int bud = static_cast<int>(budget), rec = static_cast<int>(recent);
  cudaError_t e = launch_chained(kv8_select_kernel,
                                 dim3(static_cast<unsigned>(c.H), static_cast<unsigned>(c.B)),
                                 dim3(KV8_SELECT_THREADS), 0, st, c, bud, rec, kept, lens_out);
  if (e != cudaSuccess) return cuda_status(e, "kf_kv8_evict select launch");
  const dim3 grid(static_cast<unsigned>((budget + c.P - 1) / c.P), static_cast<unsigned>(c.H),
                  static_cast<unsigned>(2 * c.B));
  const int groups = c.P * c.D / 4 / KV8_THREADS;
#define KF_KV8_MOVE(NG)                                                                        \
  e = launch_chained(kv8_move_kernel<NG>, grid, dim3(KV8_THREADS), 0, st, c, table_out, ld_out, \
                     bud, static_cast<const int32_t*>(kept))
  if (groups <= 1)
    KF_KV8_MOVE(1);
  else if (groups <= 2)
    KF_KV8_MOVE(2);
  else if (groups <= 4)
    KF_KV8_MOVE(4);
  else if (groups <= 8)
    KF_KV8_MOVE(8);
  else
    KF_KV8_MOVE(16);
#undef KF_KV8_MOVE
  return cuda_status(e, "kf_kv8_evict move launch");
}
