// Host side of kf_kv8_attention: which kernels run, how the work is cut, and
// the workspace.
#include "kv8_common.cuh"

namespace kf {

// Which kernel serves a call of `rows` query rows per kv head. Measured (us,
// split / tensor-memory kernel, at 48, 64, 96 and 128 rows): 8 x 8 heads of 128 over
// 8k tokens, bf16 107 / 138, 147 / 141, 196 / 146, 262 / 152, fp16 140 / 170, 176 / 173,
// 236 / 178, 316 / 179, fp32 133 / 162, 190 / 163, 256 / 170, 354 / 161; 16 x 12 heads of
// 64 over 1k, bf16 52 / 56, 41 / 56, 54 / 57, 72 / 56, fp32 60 / 81, 50 / 82, 65 / 83, 88 /
// 82; 8 heads of 64 over 16k, bf16 27 / 47, 33 / 47, 42 / 50, 51 / 51. The two cross
// between 48 and 64 rows at head_dim 128 and between 96 and 128 at 64; one
// threshold serves both, so 65 to about 110 rows at 64 lose up to a fifth. With weights the split kernel keeps every score for the last
// pass; where that takes too much memory (512 MB for 17 rows and more, 4 GB for
// fewer), the call goes to the other kernel, which computes the scores again.
// Few rows gain from the scores as long as they can: one token of 64 sequences of
// 4096, 8 kv heads of 128, 8 rows each, takes 331 us with 2.1 GB of scores (a
// table that reaches 131k tokens), 3625 without, and 165 us, either way, when
// max_len tells the sequences' length.
static bool kv8_is_prompt(const KV8& c, int64_t rows, int64_t max_len, int flags) {
  if (rows > KV8_SPLIT_ROWS) return true;
  const int64_t scores = static_cast<int64_t>(c.B) * c.H * rows * max_len * 4;
  return (flags & KF_KV8_TRACK) && scores > (rows > KV8_ROWS ? 512LL << 20 : 4LL << 30);
}

// How a call is cut: chunks of keys so that there are a few CTAs per SM, each
// with work enough to pay for its start.
static void kv8_plan(const KV8& c, int dtype, int64_t T, int G, int64_t max_len, int flags,
                     KV8Work* w) {
  const int64_t rows = T * G;
  w->prompt = kv8_is_prompt(c, rows, max_len, flags);
  if (w->prompt) {
    // One CTA per SM: as many parts of the keys as make the waves of CTAs cost
    // least, in steps of 128 keys. A CTA's start and end cost about four steps,
    // a part's share of the join about one. (8 heads of 128, a chunk of 1000 over 62k
    // tokens: 32 CTAs a part, 5 parts 575 us, 10 parts 472, 14 parts 423.)
    const int64_t tile = 128 * (c.D == 128 && dtype == KF_DT_F32 ? 1 : 2);
    const int64_t ctas = (rows + tile - 1) / tile * c.B * c.H;
    const int64_t steps = (max_len + 127) / 128;
    const int sms = sm_count();
    int64_t chunks = 1, best = INT64_MAX;
    for (int64_t n = 1; n <= 64 && n * 16 <= steps + 15; ++n) {
      const int64_t cost = (ctas * n + sms - 1) / sms * ((steps + n - 1) / n + 4) + n - 1;
      if (cost < best) {
        best = cost;
        chunks = n;
      }
    }
    const int64_t chunk = ((max_len + chunks - 1) / chunks + 127) / 128 * 128;
    w->chunk = static_cast<int>(chunk < 128 ? 128 : chunk);
    w->chunks = static_cast<int>((max_len + w->chunk - 1) / w->chunk);
    if (w->chunks < 1) w->chunks = 1;
    w->rows = static_cast<int>(rows);
    w->ld_score = 0;
    return;
  }
  const int64_t tiles = (rows + KV8_ROWS - 1) / KV8_ROWS;
  const int64_t items = tiles * c.B * c.H;
  // One wave of the CTAs that an SM holds. (A 65k sequence of 16 heads of 64: 42
  // us with four CTAs an SM, 50 with eight; 16 long sequences of 8 heads of 128:
  // 146 with three, 164 with eight. More parts also make the join longer.)
  const int64_t want =
      static_cast<int64_t>(sm_count()) *
      (c.D == 128 ? SplitCfg<128>::min_blocks(dtype == KF_DT_F32 ? 2 : 1) : SplitCfg<64>::min_blocks(1));
  int64_t chunks = (want + items - 1) / items;
  const int64_t most = (max_len + 127) / 128;    // at least 128 keys a chunk
  if (chunks > most) chunks = most;
  const int64_t least = (max_len + KV8_CHUNK_MAX - 1) / KV8_CHUNK_MAX;
  if (chunks < least) chunks = least;
  if (chunks < 1) chunks = 1;
  int64_t chunk = (max_len + chunks - 1) / chunks;
  chunk = (chunk + 127) / 128 * 128;             // whole pages, whatever the page
  if (chunk < 128) chunk = 128;
  w->chunk = static_cast<int>(chunk);
  w->chunks = static_cast<int>((max_len + chunk - 1) / chunk);
  if (w->chunks < 1) w->chunks = 1;
  w->rows = static_cast<int>(rows);
  w->ld_score = (flags & KF_KV8_TRACK) ? (max_len + 15) / 16 * 16 : 0;
}

// Splits the workspace; returns the bytes it takes.
static int64_t kv8_carve(const KV8& c, int dtype, int flags, uint8_t* base, KV8Work* w) {
  int64_t at = 0;
  auto take = [&](int64_t floats) -> float* {
    float* p = reinterpret_cast<float*>(base + at);
    at += (floats * 4 + 255) / 256 * 256;
    return p;
  };
  const int64_t n = static_cast<int64_t>(c.B) * c.H * w->rows;
  w->ref = w->sum = w->part = w->lse = w->score = nullptr;
  if (w->chunks > 1) {
    w->ref = take(n * w->chunks);
    w->sum = take(n * w->chunks);
    w->part = take(n * w->chunks * c.D);
  }
  if (flags & KF_KV8_TRACK) w->lse = take(n);
  if (w->ld_score) w->score = take(n * w->ld_score);
  w->planes = nullptr;
  w->qf = nullptr;
  if (w->prompt) {
    const int64_t planes = dtype == KF_DT_F32 ? 2 : 1;
    w->planes = reinterpret_cast<uint16_t*>(take((planes * n * c.D + 1) / 2));
    w->qf = take(n);
  }
  return at;
}

static int kv8_attention_check(const char* what, const kf_kv8_cache* cache, int dtype, int64_t T,
                               int64_t q_heads, int64_t* max_len, float sm_scale, int flags, KV8* c) {
  int rc = kv8_view(what, cache, c);
  if (!rc) rc = kv8_dtype(what, dtype);
  if (rc) return rc;
  if (!(sm_scale >= 0.f) || sm_scale > 3.0e38f) {
    set_last_error("%s: sm_scale must be finite and not negative", what);
    return KF_E_INVALID;
  }
  if (T < 0 || q_heads <= 0 || q_heads % c->H || (flags & ~(KF_KV8_CAUSAL | KF_KV8_TRACK)) ||
      *max_len < 0) {
    set_last_error("%s: needs T >= 0, q_heads a multiple of kv_heads and known flags", what);
    return KF_E_INVALID;
  }
  if ((flags & KF_KV8_TRACK) && c->pages && !c->weight) {
    set_last_error("%s: KF_KV8_TRACK needs a cache with a weight record", what);
    return KF_E_INVALID;
  }
  const int64_t reach = static_cast<int64_t>(c->blocks) * c->P;
  if (*max_len == 0 || *max_len > reach) *max_len = reach;
  if (static_cast<int64_t>(c->B) * c->H > 65535 || T * (q_heads / c->H) > 65535LL * KV8_ROWS) {
    set_last_error("%s: needs batch * kv_heads <= 65535 and at most 2^20 query rows a kv head",
                   what);
    return KF_E_UNSUPPORTED;
  }
  return KF_OK;
}

// Arguments of a call, for the kernels' launchers.
struct KV8Call {
  const void* q;
  int64_t q_sb, q_sh, q_st;
  void* out;
  int64_t o_sb, o_sh, o_st;
  int dtype, q_vec, q_vec16, o_vec;  // alignment: runs of 4 of q, 16 bytes of q and of out
  const int32_t* counts;
  int T, G, max_len;
  float scale_log2;
  int flags;
  float* lse;
  cudaStream_t st;
};

template <int DH, int FMT, int QP, int PP, int RH>
static cudaError_t kv8_split(const KV8& c, const KV8Call& a, const KV8Work& w) {
  auto kern = kv8_split_kernel<DH, FMT, QP, PP, RH>;
  constexpr int smem = SplitCfg<DH>::SMEM;
  static DeviceOnce once;
  cudaError_t attr = cudaSuccess;
  once.run("kf_kv8_attention", nullptr, [&](int) {
    attr = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    return attr == cudaSuccess ? KF_OK : KF_E_CUDA;
  });
  if (attr != cudaSuccess) return attr;
  const dim3 grid(static_cast<unsigned>(w.chunks),
                  static_cast<unsigned>((w.rows + KV8_ROWS - 1) / KV8_ROWS),
                  static_cast<unsigned>(c.B * c.H));
  return launch_chained(kern, grid, dim3(128), smem, a.st, c, a.q, a.q_sb, a.q_sh, a.q_st, a.out,
                        a.o_sb, a.o_sh, a.o_st, a.dtype, a.q_vec, a.counts, a.T, a.G, a.max_len,
                        a.scale_log2, a.flags, a.lse, w);
}
template <int DH, int FMT, int QP, int PP>
static cudaError_t kv8_split_rows(const KV8& c, const KV8Call& a, const KV8Work& w, bool half) {
  return half ? kv8_split<DH, FMT, QP, PP, 1>(c, a, w) : kv8_split<DH, FMT, QP, PP, 2>(c, a, w);
}
// fp16 outputs show one plane's rounding of P (1.4 times their own error), bf16
// ones do not. The second plane costs (us, one / two): a token of 4 rows a kv
// head, 24k tokens of 128, 147 / 148; of 12 rows 168 / 205; a chunk of 1024 over
// 8k tokens of 64 246 / 436 (P then takes the place of S), prompts of 2048 tokens of
// 128 288 / 380.
template <int DH, int FMT>
static cudaError_t kv8_split_type(const KV8& c, const KV8Call& a, const KV8Work& w, bool half) {
  if (a.dtype == KF_DT_F32) return kv8_split_rows<DH, FMT, 2, 2>(c, a, w, half);
  if (a.dtype == KF_DT_F16) return kv8_split_rows<DH, FMT, 1, 2>(c, a, w, half);
  return kv8_split_rows<DH, FMT, 1, 1>(c, a, w, half);
}
template <int DH>
static cudaError_t kv8_split_any(const KV8& c, const KV8Call& a, const KV8Work& w, bool half) {
  return c.fmt == KF_KV8_INT8 ? kv8_split_type<DH, KF_KV8_INT8>(c, a, w, half)
                              : kv8_split_type<DH, KF_KV8_E4M3>(c, a, w, half);
}

template <int DH, int QP, int PP>
static int kv8_prompt(const KV8& c, const KV8Call& a, const KV8Work& w) {
  using Cfg = PromptCfg<DH, QP, PP>;
  using Wei = WeighCfg<DH, QP>;
  const unsigned bh = static_cast<unsigned>(c.B * c.H);
  const bool track = (a.flags & KF_KV8_TRACK) != 0;
  CUtensorMap map;
  const uint64_t dims[3] = {DH, static_cast<uint64_t>(w.rows), static_cast<uint64_t>(QP) * bh};
  const uint64_t strides[2] = {DH * 2, static_cast<uint64_t>(w.rows) * DH * 2};
  const uint32_t box[3] = {64, 128, 1};
  int rc = encode_tensor_map(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, w.planes, dims, strides, box,
                             CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  auto kern = kv8_prompt_kernel<DH, QP, PP>;
  auto kern_w = kv8_prompt_weights_kernel<DH, QP>;
  static DeviceOnce once;
  rc = once.run("kf_kv8_attention", nullptr, [&](int) {
    cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kern_w, cudaFuncAttributeMaxDynamicSharedMemorySize, Wei::SMEM);
    return cuda_status(e, "kf_kv8_attention: set smem attribute");
  });
  if (rc) return rc;
  auto prep = a.dtype == KF_DT_F32    ? kv8_prep_q_kernel<KF_DT_F32>
              : a.dtype == KF_DT_BF16 ? kv8_prep_q_kernel<KF_DT_BF16>
                                      : kv8_prep_q_kernel<KF_DT_F16>;
  const int rows_of_cta = 256 * (QP == 2 ? 4 : 8) / DH * KV8_PREP_UNROLL;
  cudaError_t e = launch_chained(
      prep, dim3(static_cast<unsigned>((w.rows + rows_of_cta - 1) / rows_of_cta), bh), dim3(256), 0,
      a.st, c, a.q, a.q_sb, a.q_sh, a.q_st, a.q_vec16, a.counts, a.T, a.G, a.scale_log2, w);
  if (e == cudaSuccess)
    e = launch_chained(kern,
                       dim3(static_cast<unsigned>((w.rows + Cfg::ROWS - 1) / Cfg::ROWS),
                            static_cast<unsigned>(w.chunks), bh),
                       dim3(Cfg::THREADS), Cfg::SMEM, a.st, map, c, a.out, a.o_sb, a.o_sh, a.o_st,
                       a.dtype, a.o_vec, a.counts, a.T, a.G, a.max_len, a.flags, a.lse, w);
  if (e == cudaSuccess && w.chunks > 1)
    e = launch_chained(kv8_join_kernel, dim3(static_cast<unsigned>(w.rows), bh), dim3(KV8_JOIN_THREADS), 0, a.st,
                       c, a.out, a.o_sb, a.o_sh, a.o_st, a.dtype, a.T, a.G, a.lse, w);
  if (e == cudaSuccess && track && a.max_len > 0)
    e = launch_chained(kern_w, dim3(static_cast<unsigned>((a.max_len + 127) / 128), bh),
                       dim3(Wei::THREADS), Wei::SMEM, a.st, map, c, a.counts, a.T, a.G, a.max_len,
                       a.flags, w);
  return cuda_status(e, "kf_kv8_attention launch");
}

template <int DH>
static int kv8_prompt_type(const KV8& c, const KV8Call& a, const KV8Work& w) {
  if (a.dtype == KF_DT_F32) return kv8_prompt<DH, 2, 2>(c, a, w);
  if (a.dtype == KF_DT_F16) return kv8_prompt<DH, 1, 2>(c, a, w);
  return kv8_prompt<DH, 1, 1>(c, a, w);
}

}  // namespace kf

using namespace kf;

extern "C" int64_t kf_kv8_attention_workspace_bytes(const kf_kv8_cache* cache, int dtype,
                                                    int64_t T, int64_t q_heads, int64_t max_len,
                                                    int flags) {
  KV8 c;
  if (kv8_attention_check("kf_kv8_attention_workspace_bytes", cache, dtype, T, q_heads, &max_len, 1.f,
                          flags, &c))
    return -1;
  if (T == 0 || c.B == 0) return 0;
  KV8Work w;
  kv8_plan(c, dtype, T, static_cast<int>(q_heads / c.H), max_len, flags, &w);
  return kv8_carve(c, dtype, flags, nullptr, &w);
}

extern "C" int kf_kv8_attention(const kf_kv8_cache* cache, const void* q, int64_t q_sb,
                                int64_t q_sh, int64_t q_st, void* out, int64_t o_sb, int64_t o_sh,
                                int64_t o_st, int dtype, const int32_t* counts, int64_t T,
                                int64_t q_heads, int64_t max_len, float sm_scale, int flags,
                                float* lse, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  KV8 c;
  int rc = kv8_attention_check("kf_kv8_attention", cache, dtype, T, q_heads, &max_len, sm_scale,
                               flags, &c);
  if (rc) return rc;
  if (T == 0 || c.B == 0) return KF_OK;
  if (!q || !out) {
    set_last_error("kf_kv8_attention: q and out must not be null");
    return KF_E_INVALID;
  }
  const int G = static_cast<int>(q_heads / c.H);
  KV8Work w;
  kv8_plan(c, dtype, T, G, max_len, flags, &w);
  const int64_t need = kv8_carve(c, dtype, flags, static_cast<uint8_t*>(workspace), &w);
  if (need > 0 && (!workspace || workspace_bytes < need || !kv8_aligned(workspace, 256))) {
    set_last_error("kf_kv8_attention: needs a 256-byte aligned workspace of %lld bytes",
                   (long long)need);
    return KF_E_INVALID;
  }
  const int64_t es = dtype_size(dtype);
  const int vec = kv8_aligned(q, 4 * es) && q_sb % 4 == 0 && q_sh % 4 == 0 && q_st % 4 == 0;
  const float scale_log2 = sm_scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int Ti = static_cast<int>(T), cap = static_cast<int>(max_len);
  const unsigned bh = static_cast<unsigned>(c.B * c.H);
  const int64_t per = 16 / es;
  const int o_vec = kv8_aligned(out, 16) && o_sb % per == 0 && o_sh % per == 0 && o_st % per == 0;
  const int vec16 = kv8_aligned(q, 16) && q_sb % per == 0 && q_sh % per == 0 && q_st % per == 0;
  const KV8Call a = {q, q_sb, q_sh, q_st, out, o_sb, o_sh, o_st, dtype, vec, vec16, o_vec, counts, Ti, G,
                     cap, scale_log2, flags, lse, st};
  if (w.prompt) {
    switch (c.D) {
      case 16: return kv8_prompt_type<16>(c, a, w);
      case 32: return kv8_prompt_type<32>(c, a, w);
      case 64: return kv8_prompt_type<64>(c, a, w);
      default: return kv8_prompt_type<128>(c, a, w);
    }
  }
  cudaError_t e = cudaSuccess;
  const bool half = w.rows <= 8;
  switch (c.D) {
    case 16: e = kv8_split_any<16>(c, a, w, half); break;
    case 32: e = kv8_split_any<32>(c, a, w, half); break;
    case 64: e = kv8_split_any<64>(c, a, w, half); break;
    default: e = kv8_split_any<128>(c, a, w, half); break;
  }
  if (e != cudaSuccess) return cuda_status(e, "kf_kv8_attention launch");
  if (w.chunks > 1) {
    e = launch_chained(kv8_join_kernel, dim3(static_cast<unsigned>(w.rows), bh), dim3(KV8_JOIN_THREADS), 0, st,
                       c, out, o_sb, o_sh, o_st, dtype, Ti, G, lse, w);
    if (e != cudaSuccess) return cuda_status(e, "kf_kv8_attention join launch");
  }
  if (max_len == 0 || !(flags & KF_KV8_TRACK)) return KF_OK;
  e = launch_chained(
      kv8_weights_kernel,
      dim3(static_cast<unsigned>((max_len + KV8_WEIGHTS_KEYS - 1) / KV8_WEIGHTS_KEYS), bh),
      dim3(128), 0, st, c, counts, Ti, G, cap, flags, w);
  return cuda_status(e, "kf_kv8_attention weights launch");
}
