// Attention of many query rows (prompt chunks) over the 8-bit cache on the
// tcgen05 tensor cores, and the attention weights that such rows give each
// cached token.
//
// kv8_prompt_kernel: one CTA = two tiles of 128 query rows (row = token * G +
// head of the group, so the query heads of a kv head share its K and V) of one
// (sequence, kv head), over a range of keys. Roles:
//   warps 0-3, 4-7  softmax of tile 0 and 1, one thread per row: reads its S
//                   row from TMEM in halves of 64, writes P over it as fp16;
//   warps 8-11      load the codes of the next 128 keys into registers while
//                   the current ones are in use, and write them as fp16 into
//                   128-byte-swizzled tiles (K: K-major, V: MN-major, the same
//                   bytes: rows are keys); codes are exact in fp16;
//   warp 12         (of 12-15) allocates TMEM, loads Q by TMA and issues the products
//                   S = Q K^T (operands in shared memory) and O += P V (P read
//                   from TMEM).
// TMEM: S0 | S1 (128 columns each, P in place), O0 | O1. For each tile the
// order is P V(j), then S(j + 1): the pipe runs in issue order, so a softmax
// that sees S(j + 1) knows O holds P V(j) and may rescale it at once, and while
// one tile's products run the other tile's softmax has the exponential unit.
// What bounds it: the exponentials, 16 a clock and SM: 2048 clocks for two
// tiles against 128 keys, where the products take 1024 at head_dim 64.
//
// Numbers as in the split kernel: q rows scaled by powers of two and P relative
// to a lazily moved reference, one fp16 plane for 16-bit q and two for fp32 q
// (then both products run twice); page scales enter S exactly and P as the
// ratio to the range's largest V scale.
//
// kv8_prompt_weights_kernel: one CTA = 128 keys against all rows that see
// them: S^T = K Q^T puts a key in each TMEM lane, so a thread adds its key's
// weights in a register over every row, in a fixed order and without atomics.
#include "kv8_common.cuh"

namespace kf {

// Instruction descriptor for kind::f16 with F16 A/B and an FP32 accumulator.
__host__ __device__ constexpr uint32_t make_idesc_f16(int M, int N, int b_mn_major) {
  return (1u << 4) | (static_cast<uint32_t>(b_mn_major) << 16) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// D[tmem] (+)= A[tmem] * B[smem], F16 inputs, FP32 accumulate.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Registers a thread of this warpgroup may use from here on (all of its warps
// execute it).
template <bool INC, int N>
__device__ __forceinline__ void set_max_registers() {
  if constexpr (INC)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  else
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// ---------------------------------------------------------------- q planes

// q rows as fp16 planes [PL][B*H][rows][D] and their factors to log2 units.
// Four lanes a row. Rows past a sequence's count get zeros.
template <int DH, int PL>
__global__ void __launch_bounds__(256)
    kv8_prep_q_kernel(KV8 c, const void* __restrict__ q, int64_t q_sb, int64_t q_sh, int64_t q_st,
                      int dtype, int vec, const int32_t* __restrict__ counts, int T, int G,
                      float scale_log2, KV8Work w) {
  const int rows = w.rows;
  uint16_t* planes = w.planes;
  float* qf = w.qf;
  pdl_launch_dependents();
  pdl_wait();
  constexpr int E = DH / 4;
  const int row = blockIdx.x * 64 + (threadIdx.x >> 2);
  const int t = threadIdx.x & 3;
  const int bh = blockIdx.y;
  const int b = bh / c.H, h = bh - b * c.H;
  const int tok = row / G;
  const bool real = row < rows && tok < kv8_count(counts, b, T);
  float x[E];
  float amax = 0.f;
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    float y[4] = {0.f, 0.f, 0.f, 0.f};
    if (real)
      kv8_load4(q, b * q_sb + static_cast<int64_t>(h * G + row - tok * G) * q_sh + tok * q_st +
                       t * E + e, dtype, vec != 0, y);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      x[e + u] = y[u];
      amax = __uint_as_float(max(__float_as_uint(amax), __float_as_uint(fabsf(y[u]))));
    }
  }
#pragma unroll
  for (int d = 1; d <= 2; d <<= 1)
    amax = __uint_as_float(
        max(__float_as_uint(amax), __shfl_xor_sync(0xffffffffu, __float_as_uint(amax), d)));
  if (row >= rows) return;
  float inv;
  const float sc = kv8_row_scale(amax, &inv);
  const int64_t at = (static_cast<int64_t>(bh) * rows + row) * DH + t * E;
  const int64_t plane = static_cast<int64_t>(c.B) * c.H * rows * DH;
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const uint32_t h0 = pack_half2(x[e] * sc, x[e + 1] * sc);
    const uint32_t h1 = pack_half2(x[e + 2] * sc, x[e + 3] * sc);
    *reinterpret_cast<uint2*>(planes + at + e) = make_uint2(h0, h1);
    if constexpr (PL == 2)
      *reinterpret_cast<uint2*>(planes + plane + at + e) =
          make_uint2(pack_half2_rest(x[e] * sc, x[e + 1] * sc, h0),
                     pack_half2_rest(x[e + 2] * sc, x[e + 3] * sc, h1));
  }
  if (t == 0) qf[static_cast<int64_t>(bh) * rows + row] = real ? inv * scale_log2 : 0.f;
}

// ---------------------------------------------------------------- tiles

// 16 codes to 16 fp16 values in a 128-byte-swizzled tile: row r, columns
// 16 * c16 .. + 15 of a 64-column half (chunk blocks of `rows` rows).
__device__ __forceinline__ void kv8_put16(uint8_t* tile, int rows, int r, int c16, uint4 w,
                                          int fmt) {
  uint32_t h[8];
  if (fmt == KF_KV8_INT8) {
    kv8_cvt4<KF_KV8_INT8>(w.x, h[0], h[1]);
    kv8_cvt4<KF_KV8_INT8>(w.y, h[2], h[3]);
    kv8_cvt4<KF_KV8_INT8>(w.z, h[4], h[5]);
    kv8_cvt4<KF_KV8_INT8>(w.w, h[6], h[7]);
  } else {
    kv8_cvt4<KF_KV8_E4M3>(w.x, h[0], h[1]);
    kv8_cvt4<KF_KV8_E4M3>(w.y, h[2], h[3]);
    kv8_cvt4<KF_KV8_E4M3>(w.z, h[4], h[5]);
    kv8_cvt4<KF_KV8_E4M3>(w.w, h[6], h[7]);
  }
  uint8_t* row = tile + (c16 >> 2) * rows * 128 + r * 128;
  const int ch = (c16 & 3) * 2;
  *reinterpret_cast<uint4*>(row + (((ch) ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
  *reinterpret_cast<uint4*>(row + (((ch + 1) ^ (r & 7)) << 4)) =
      make_uint4(h[4], h[5], h[6], h[7]);
}

// N consecutive outputs of one row; `vec`: 16-byte aligned.
template <int N>
__device__ __forceinline__ void kv8_store_run(void* out, int64_t at, int dtype, bool vec,
                                              const float* o) {
  if (!vec) {
#pragma unroll
    for (int u = 0; u < N; ++u) kv8_store1(out, at + u, dtype, o[u]);
  } else if (dtype == KF_DT_F32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
#pragma unroll
    for (int u = 0; u < N; u += 4) p[u >> 2] = make_float4(o[u], o[u + 1], o[u + 2], o[u + 3]);
  } else {
    uint4* p = reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at);
#pragma unroll
    for (int u = 0; u < N; u += 8) {
      uint32_t x[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        if (dtype == KF_DT_BF16) {
          const __nv_bfloat162 y = __floats2bfloat162_rn(o[u + 2 * v], o[u + 2 * v + 1]);
          x[v] = *reinterpret_cast<const uint32_t*>(&y);
        } else {
          x[v] = pack_half2(o[u + 2 * v], o[u + 2 * v + 1]);
        }
      }
      p[u >> 3] = make_uint4(x[0], x[1], x[2], x[3]);
    }
  }
}

template <int DH, int PL>
struct PromptCfg {
  static constexpr int BM = 128;                           // query rows of a tile
  static constexpr int BN = (DH == 128 && PL == 2) ? 64 : 128;  // keys of a step
  static constexpr int CH = DH > 64 ? 2 : 1;               // 64-column halves of a row
  static constexpr int Q_PLANE = BM * 128 * CH;            // bytes of one tile's plane
  static constexpr int Q_BYTES = 2 * PL * Q_PLANE;
  static constexpr int KV_BYTES = BN * 128 * CH;
  static constexpr int ST = 2;                             // stages of K and of V
  static constexpr int K_OFF = Q_BYTES;
  static constexpr int V_OFF = K_OFF + ST * KV_BYTES;
  static constexpr int BAR_OFF = V_OFF + ST * KV_BYTES;
  static constexpr int SC_OFF = BAR_OFF + 256;             // page scales of each stage
  // Four slots, each read by step j's softmax and rewritten for step j + 4: by
  // then every softmax warp has begun step j + 2.
  static constexpr int SLOTS = 4;
  static constexpr int USED = SC_OFF + SLOTS * 128 + 1024;
  // One CTA per SM (all of TMEM): ask for more than half of shared memory.
  static constexpr int SMEM = USED > 120 * 1024 ? USED : 120 * 1024;
  static constexpr int GROUPS = BN / 16;                   // scale entries of a stage
  static constexpr int LOADS = BN * DH / 16 / 128;         // 16-byte loads a loader thread
  static constexpr int O_COL = 256;
  static constexpr int O_STRIDE = DH < 32 ? 32 : DH;       // columns between O0 and O1
  // Four warpgroups launched with 128 registers a thread; the softmax ones
  // take 176 (a row of 64 scores and its packed P), the loaders keep 96, the
  // issuer's 64: 8 * 176 + 4 * 96 + 4 * 64 = 16 * 128.
  static constexpr int THREADS = 16 * 32;
  static_assert(SMEM <= 232448, "smem");
  static_assert(O_COL + 2 * O_STRIDE <= 512, "TMEM");
};

// Scales of the keys of one stage, by groups of 16 keys.
struct alignas(16) PromptScales {
  float ks[8];
  float ratio[8];   // V scale over the range's largest
  uint32_t bad;      // groups on a refused page
  uint32_t spoiled;  // groups on a page whose V scale is NaN (their ratio is 0)
};

// One row's 64 scores of a half tile: loaded, scaled to log2 units, masked.
template <int BN>
__device__ __forceinline__ void prompt_scores(uint32_t t_addr, float qf, const float* ks,
                                              uint32_t bad, bool mask, int limit, float (&s)[64]) {
  tmem_ld64(t_addr, s);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const float f = qf * ks[g];
    const uint64_t f2 = f2_pack(f, f);
#pragma unroll
    for (int u = 0; u < 16; u += 2)
      f2_unpack(f2_mul(f2_pack(s[16 * g + u], s[16 * g + u + 1]), f2), s[16 * g + u],
                s[16 * g + u + 1]);
  }
  if (mask) {
    uint32_t kw[2];
#pragma unroll
    for (int w = 0; w < 2; ++w)
      kw[w] = ((bad >> (2 * w)) & 1u ? 0u : 0x0000ffffu) |
              ((bad >> (2 * w + 1)) & 1u ? 0u : 0xffff0000u);
    mask_scores<64>(s, kw, limit);
  }
}

__device__ __forceinline__ float max64(const float (&s)[64]) {
  float m[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) m[u] = fmaxf(s[u], s[u + 8]);
#pragma unroll
  for (int c = 16; c < 64; c += 16) {
#pragma unroll
    for (int u = 0; u < 8; ++u) m[u] = fmax3(m[u], s[c + u], s[c + 8 + u]);
  }
  return fmax3(fmax3(m[0], m[1], m[2]), fmax3(m[3], m[4], m[5]), fmaxf(m[6], m[7]));
}

// Store 16 consecutive TMEM columns of this thread's lane (no wait).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// P of 64 scores: fp16 words (and the second plane's), the unrounded sum.
template <int PL>
__device__ __forceinline__ float prompt_weights(const float (&s)[64], float neg_ref,
                                                const float* ratio, uint32_t t_addr) {
  uint64_t acc[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
  const uint64_t nr = f2_pack(neg_ref, neg_ref);
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int k = 32 * part + 2 * u;
      float a, b;
      f2_unpack(f2_add(f2_pack(s[k], s[k + 1]), nr), a, b);
      a = fast_exp2(a);
      b = fast_exp2(b);
      acc[u & 1] = f2_add(acc[u & 1], f2_pack(a, b));
      const float r = ratio[k >> 4];
      f2_unpack(f2_mul(f2_pack(a, b), f2_pack(r, r)), a, b);
      hi[u] = pack_half2(a, b);
      if constexpr (PL == 2) lo[u] = pack_half2_rest(a, b, hi[u]);
    }
    tmem_st16(t_addr + 16 * part, hi);
    if constexpr (PL == 2) tmem_st16(t_addr + 32 + 16 * part, lo);
  }
  float x0, x1, x2, x3;
  f2_unpack(acc[0], x0, x1);
  f2_unpack(acc[1], x2, x3);
  return (x0 + x1) + (x2 + x3);
}

template <int DH, int PL>
__global__ void __launch_bounds__(PromptCfg<DH, PL>::THREADS, 1)
    kv8_prompt_kernel(const __grid_constant__ CUtensorMap tmQ, KV8 c, void* __restrict__ out,
                      int64_t o_sb, int64_t o_sh, int64_t o_st, int dtype, int o_vec,
                      const int32_t* __restrict__ counts, int T, int G, int max_len, int flags,
                      float* __restrict__ lse_out, KV8Work w) {
  using Cfg = PromptCfg<DH, PL>;
  constexpr int BM = Cfg::BM, BN = Cfg::BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + Cfg::K_OFF;
  uint8_t* sV = smem + Cfg::V_OFF;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;    // [ST] 4 loader warps
  uint64_t* v_full = bars + 3;    // [ST]
  uint64_t* k_empty = bars + 5;   // [ST] S of both tiles done, 8 softmax warps at that step
  uint64_t* v_empty = bars + 7;   // [ST] P V of both tiles done
  uint64_t* s_full = bars + 9;    // [2]
  uint64_t* p_full = bars + 11;   // [2] 4 warps
  uint64_t* o_final = bars + 13;  // [2]
  uint64_t* drain = bars + 15;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_vmax = reinterpret_cast<float*>(tmem_slot + 2);  // [16]
  PromptScales* s_sc = reinterpret_cast<PromptScales*>(smem + Cfg::SC_OFF);
  static_assert(sizeof(PromptScales) <= 128, "scale ring");

  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bh = blockIdx.z;
  const int b = bh / c.H, h = bh - b * c.H;
  const int chunk = blockIdx.y;
  const int row0 = static_cast<int>(gridDim.x - 1 - blockIdx.x) * 2 * BM;  // heaviest first
  const int len = kv8_len(c, b);
  const int count = kv8_count(counts, b, T);
  int end = kv8_end(c, len, count);
  if (end > max_len) {
    if (tid == 0) record_device_status(KF_DEV_BAD_KV_PAGE);
    end = max_len;
  }
  const bool causal = (flags & KF_KV8_CAUSAL) != 0;
  const int last_row = min(row0 + 2 * BM, w.rows) - 1;
  const int last_tok = min(last_row / G, count - 1);
  const int reach = last_tok < row0 / G ? 0 : (causal ? min(len + last_tok + 1, end) : end);
  const int k0 = chunk * w.chunk;
  const int k1 = min(k0 + w.chunk, reach);
  const bool alone = w.chunks == 1;
  if (k0 >= k1) {
    // No key: zeros, or an empty part for the join.
    for (int i = tid; i < 2 * BM; i += Cfg::THREADS) {
      const int row = row0 + i;
      if (row >= w.rows) break;
      const int64_t at = static_cast<int64_t>(bh) * w.rows + row;
      if (!alone) {
        w.ref[at * w.chunks + chunk] = -INFINITY;
        w.sum[at * w.chunks + chunk] = 0.f;
        continue;
      }
      const int tok = row / G, hq = h * G + row - tok * G;
      for (int d = 0; d < DH; ++d) kv8_store1(out, b * o_sb + hq * o_sh + tok * o_st + d, dtype, 0.f);
      if (lse_out) lse_out[(static_cast<int64_t>(b) * c.H * G + hq) * T + tok] = -INFINITY;
      if (w.lse) w.lse[at] = -INFINITY;
    }
    return;
  }
  const int n_steps = (k1 - k0 + BN - 1) / BN;

  if (tid == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&v_full[s], 4);
      mbar_init(&k_empty[s], 1 + 8);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&o_final[s], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
  }
  if (warp == 12) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // The largest V scale of the range.
  {
    float vmax = 0.f;
    for (int j = (k0 >> c.p_shift) + tid; (j << c.p_shift) < k1; j += Cfg::THREADS) {
      const int page = kv8_page(c, b, j);
      if (page >= 0) vmax = fmaxf(vmax, __ldg(c.scale + 2 * (static_cast<int64_t>(page) * c.H + h) + 1));
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, d));
    if (lane == 0) s_vmax[warp] = vmax;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();  // every CTA that runs holds its TMEM by now
  float vmax = s_vmax[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) vmax = fmaxf(vmax, s_vmax[i]);

  if (warp >= 12) {
    set_max_registers<false, 64>();
    if (warp == 12 && lane == 0) {
      // ------------------------------------------------ Q, products
      mbar_arrive_expect_tx(q_full, Cfg::Q_BYTES);
      for (int t = 0; t < 2; ++t)
        for (int pl = 0; pl < PL; ++pl)
          for (int ch = 0; ch < Cfg::CH; ++ch)
            tma_load_3d(sQ + (t * PL + pl) * Cfg::Q_PLANE + ch * BM * 128, &tmQ, q_full, ch * 64,
                        row0 + t * BM, pl * c.B * c.H + bh);
      constexpr uint32_t idesc_s = make_idesc_f16(BM, BN, 0);
      constexpr uint32_t idesc_o = make_idesc_f16(BM, DH, 1);
      const uint32_t sQa = smem_u32(sQ), sKa = smem_u32(sK), sVa = smem_u32(sV);
      auto issue_s = [&](int t, int stage) {
#pragma unroll
        for (int pl = PL - 1; pl >= 0; --pl)  // the small plane first
#pragma unroll
          for (int kk = 0; kk < DH / 16; ++kk) {
            const uint64_t ad = make_smem_desc(sQa + (t * PL + pl) * Cfg::Q_PLANE +
                                                   (kk >> 2) * BM * 128 + (kk & 3) * 32,
                                               16, 1024, KF_SWIZZLE_128B);
            const uint64_t bd =
                make_smem_desc(sKa + stage * Cfg::KV_BYTES + (kk >> 2) * BN * 128 + (kk & 3) * 32,
                               16, 1024, KF_SWIZZLE_128B);
            mma_bf16_ss(tmem_base + t * 128, ad, bd, idesc_s, (pl < PL - 1 || kk > 0) ? 1u : 0u);
          }
        mma_commit(&s_full[t]);
      };
      bool ok = mbar_wait(q_full, 0, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA) &&
                mbar_wait(&k_full[0], 0, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA);
      if (ok) {
        tc_fence_after();
        issue_s(0, 0);
        issue_s(1, 0);
        mma_commit(&k_empty[0]);
      }
      for (int j = 0; j < n_steps && ok; ++j) {
        const int st = j & 1, nx = (j + 1) & 1;
        const uint32_t ph = (j >> 1) & 1, nph = ((j + 1) >> 1) & 1;
        ok = mbar_wait(&v_full[st], ph, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA);
        for (int t = 0; t < 2 && ok; ++t) {
          ok = mbar_wait(&p_full[t], j & 1, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int pl = PL - 1; pl >= 0; --pl)
#pragma unroll
            for (int kk = 0; kk < BN / 16; ++kk) {
              const uint64_t bd = make_smem_desc(sVa + st * Cfg::KV_BYTES + kk * 16 * 128, BN * 128,
                                                 1024, KF_SWIZZLE_128B);
              mma_f16_ts(tmem_base + Cfg::O_COL + t * Cfg::O_STRIDE,
                         tmem_base + t * 128 + (kk >> 2) * 64 + pl * 32 + (kk & 3) * 8, bd,
                         idesc_o, (j > 0 || pl < PL - 1 || kk > 0) ? 1u : 0u);
            }
          if (j + 1 < n_steps) {
            if (t == 0) {
              ok = mbar_wait(&k_full[nx], nph, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA);
              if (!ok) break;
              tc_fence_after();
            }
            issue_s(t, nx);
          } else {
            mma_commit(&o_final[t]);
          }
        }
        if (ok) {
          mma_commit(&v_empty[st]);
          if (j + 1 < n_steps) mma_commit(&k_empty[nx]);
        }
      }
      mma_commit(drain);
      mbar_wait_drain(drain, 0, KF_DEV_WAIT_TIMEOUT_MMA);
      mbar_wait_drain(q_full, 0, KF_DEV_WAIT_TIMEOUT_MMA);
    }
  } else if (warp >= 8) {
    // -------------------------------------------------- loaders
    set_max_registers<false, 96>();
    const int lt = tid - 256;
    const float inv_vmax = vmax > 0.f ? 1.f / vmax : 0.f;
    constexpr int RC = DH / 16;  // 16-byte pieces of a row
    uint4 kr[Cfg::LOADS], vr[Cfg::LOADS];
    float sc_k = 0.f, sc_r = 0.f;
    bool sc_bad = false;
    auto load = [&](const uint8_t* pool, int key0, uint4 (&r)[Cfg::LOADS]) {
#pragma unroll
      for (int i = 0; i < Cfg::LOADS; ++i) {
        const int id = i * 128 + lt;
        const int key = key0 + id / RC;
        r[i] = make_uint4(0u, 0u, 0u, 0u);
        if (key < k1) {
          const int page = kv8_page(c, b, key >> c.p_shift);
          if (page >= 0)
            r[i] = __ldg(reinterpret_cast<const uint4*>(
                       pool + ((static_cast<int64_t>(page) * c.H + h) * c.P + (key & (c.P - 1))) * DH) +
                   id % RC);
        }
      }
    };
    auto put = [&](uint8_t* tile, const uint4 (&r)[Cfg::LOADS]) {
#pragma unroll
      for (int i = 0; i < Cfg::LOADS; ++i) {
        const int id = i * 128 + lt;
        kv8_put16(tile, BN, id / RC, id % RC, r[i], c.fmt);
      }
      fence_proxy_async_smem();
    };
    auto load_scale = [&](int key0) {
      if (lt >= Cfg::GROUPS) return;
      const int key = key0 + lt * 16;
      sc_k = sc_r = 0.f;
      sc_bad = false;
      if (key < k1) {
        const int page = kv8_page(c, b, key >> c.p_shift);
        sc_bad = page < 0;
        if (page >= 0) {
          const float2 s = __ldg(reinterpret_cast<const float2*>(
              c.scale + 2 * (static_cast<int64_t>(page) * c.H + h)));
          sc_k = s.x;
          sc_r = s.y * inv_vmax;
        }
      }
    };
    load_scale(k0);
    load(c.k, k0, kr);
    load(c.v, k0, vr);
    for (int j = 0; j < n_steps; ++j) {
      const int st = j & 1;
      const uint32_t eph = ((j >> 1) & 1) ^ 1;  // phase of the release two steps back
      if (j >= 2 && !mbar_wait(&k_empty[st], eph, abort_flag, KF_DEV_WAIT_TIMEOUT_TMA)) break;
      put(sK + st * Cfg::KV_BYTES, kr);
      if (lt < 32) {
        const uint32_t bad = __ballot_sync(0xffffffffu, sc_bad);
        const uint32_t spoiled = __ballot_sync(0xffffffffu, sc_r != sc_r);
        if (lt < Cfg::GROUPS) {
          s_sc[j & 3].ks[lt] = sc_k;
          s_sc[j & 3].ratio[lt] = sc_r == sc_r ? sc_r : 0.f;
        }
        if (lt == 0) {
          s_sc[j & 3].bad = bad;
          s_sc[j & 3].spoiled = spoiled;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[st]);
      const int next = k0 + (j + 1) * BN;
      if (j + 1 < n_steps) {
        load_scale(next);
        load(c.k, next, kr);
      }
      if (j >= 2 && !mbar_wait(&v_empty[st], eph, abort_flag, KF_DEV_WAIT_TIMEOUT_TMA)) break;
      put(sV + st * Cfg::KV_BYTES, vr);
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[st]);
      if (j + 1 < n_steps) load(c.v, next, vr);
    }
  } else {
    // -------------------------------------------------- softmax
    set_max_registers<true, 176>();
    const int t = warp >> 2;
    const int quarter = warp & 3;
    const int row = row0 + t * BM + quarter * 32 + lane;
    const int tok = row / G;
    const int limit = (row < w.rows && tok < count) ? (causal ? min(len + tok + 1, end) : end) : 0;
    const float qf = row < w.rows ? __ldg(w.qf + static_cast<int64_t>(bh) * w.rows + row) : 0.f;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_s = t_row + t * 128;
    const uint32_t t_o = t_row + Cfg::O_COL + t * Cfg::O_STRIDE;
    float ref = -INFINITY, sum = 0.f;
    bool ok = true, nan_row = false;
    for (int j = 0; j < n_steps; ++j) {
      const int st = j & 1;
      if (!mbar_wait(&k_full[st], (j >> 1) & 1, abort_flag, KF_DEV_WAIT_TIMEOUT_SOFTMAX) ||
          !mbar_wait(&s_full[t], j & 1, abort_flag, KF_DEV_WAIT_TIMEOUT_SOFTMAX)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (lane == 0) mbar_arrive(&k_empty[st]);
      const PromptScales& sc = s_sc[j & 3];
      const float* ks = sc.ks;
      const float* ratio = sc.ratio;
      const uint32_t bad = sc.bad;
      const uint32_t spoiled = sc.spoiled;
      const int key0 = k0 + j * BN;
      const int lim = min(limit, k1) - key0;
      const bool mask = __any_sync(0xffffffffu, lim < BN) || bad;
      // Only rows that see a token of a spoiled page are NaN: decided per row,
      // since 0 * NaN in the product would reach rows that do not.
      if (spoiled && lim > 16 * (__ffs(static_cast<int>(spoiled)) - 1)) nan_row = true;
      float s[64];
      float mx = -INFINITY;
      if constexpr (BN == 128) {
        prompt_scores<BN>(t_s, qf, ks, bad, mask, lim, s);
        mx = max64(s);
        prompt_scores<BN>(t_s + 64, qf, ks + 4, bad >> 4, mask, lim - 64, s);
      } else {
        prompt_scores<BN>(t_s, qf, ks, bad, mask, lim, s);
      }
      mx = fmaxf(mx, max64(s));
      // The reference moves when the maximum has outgrown it by more than the
      // slack. S of this step was issued after P V of the last, so O is at rest.
      float alpha = 1.f;
      const bool move = mx > ref + (KV8_BIAS + KV8_SLACK);
      if (move) {
        if (ref != -INFINITY) alpha = fast_exp2(ref - (mx - KV8_BIAS));
        ref = mx - KV8_BIAS;
        sum *= alpha;
      }
      if (j > 0 && __any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int cc = 0; cc < (DH + 31) / 32; ++cc) {
          float o[32];  // head_dim 16: the columns past O are unused
          tmem_ld32(t_o + cc * 32, o);
#pragma unroll
          for (int u = 0; u < 32; ++u) o[u] *= alpha;
          tmem_st32(t_o + cc * 32, o);
        }
      }
      const float neg = ref == -INFINITY ? 0.f : -ref;
      if constexpr (BN == 128) {
        sum += prompt_weights<PL>(s, neg, ratio + 4, t_s + 64);
        prompt_scores<BN>(t_s, qf, ks, bad, mask, lim, s);
      }
      sum += prompt_weights<PL>(s, neg, ratio, t_s);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    if (ok && mbar_wait(&o_final[t], 0, abort_flag, KF_DEV_WAIT_TIMEOUT_SOFTMAX)) {
      tc_fence_after();
      const int64_t at = static_cast<int64_t>(bh) * w.rows + row;
      const int hq = h * G + row - tok * G;
      float f = alone ? vmax / sum : vmax;  // not used where sum is 0
      if (nan_row) f = __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int cc = 0; cc < (DH + 31) / 32; ++cc) {
        float o[32];
        tmem_ld32(t_o + cc * 32, o);
        if (row >= w.rows) continue;
#pragma unroll
        for (int u = 0; u < 32; ++u) o[u] = sum == 0.f ? 0.f : o[u] * f;
        constexpr int NC = DH < 32 ? DH : 32;
        if (alone) {
          kv8_store_run<NC>(out, b * o_sb + hq * o_sh + tok * o_st + cc * 32, dtype, o_vec != 0, o);
        } else {
          float4* p = reinterpret_cast<float4*>(w.part + (at * w.chunks + chunk) * DH + cc * 32);
#pragma unroll
          for (int u = 0; u < NC; u += 4) p[u >> 2] = make_float4(o[u], o[u + 1], o[u + 2], o[u + 3]);
        }
      }
      if (row < w.rows) {
        if (alone) {
          const float l2 = sum == 0.f ? -INFINITY : ref + log2f(sum);
          if (lse_out)
            lse_out[(static_cast<int64_t>(b) * c.H * G + hq) * T + tok] = l2 * 0.6931471805599453f;
          if (w.lse) w.lse[at] = l2;
        } else {
          w.ref[at * w.chunks + chunk] = ref;
          w.sum[at * w.chunks + chunk] = sum;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) {
    __syncwarp();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- weights

template <int DH, int PL>
struct WeighCfg {
  static constexpr int BK = 128;                   // keys of a CTA (TMEM lanes)
  static constexpr int BR = 128;                   // query rows of a step
  static constexpr int CH = DH > 64 ? 2 : 1;
  static constexpr int K_BYTES = BK * 128 * CH;
  static constexpr int Q_PLANE = BR * 128 * CH;
  static constexpr int Q_STAGE = PL * Q_PLANE;
  static constexpr int ST = 2;
  static constexpr int Q_OFF = K_BYTES;
  static constexpr int ROW_OFF = Q_OFF + ST * Q_STAGE;   // factors and lse of a stage's rows
  static constexpr int BAR_OFF = ROW_OFF + ST * BR * 8;
  static constexpr int SUM_OFF = BAR_OFF + 256;
  static constexpr int SMEM = SUM_OFF + BK * 4 + 1024;
  static constexpr int THREADS = 10 * 32;
  static constexpr int LOADS = BK * DH / 16 / 256;  // by the eight adding warps
  static_assert(SMEM <= 232448, "smem");
};

template <int DH, int PL>
__global__ void __launch_bounds__(WeighCfg<DH, PL>::THREADS)
    kv8_prompt_weights_kernel(const __grid_constant__ CUtensorMap tmQ, KV8 c,
                              const int32_t* __restrict__ counts, int T, int G, int max_len,
                              int flags, KV8Work w) {
  using Cfg = WeighCfg<DH, PL>;
  constexpr int BR = Cfg::BR;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sK = smem;
  uint8_t* sQ = smem + Cfg::Q_OFF;
  float* s_row = reinterpret_cast<float*>(smem + Cfg::ROW_OFF);  // [ST][2][BR]: factor, -lse
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::BAR_OFF);
  uint64_t* q_full = bars;       // [ST] TMA bytes
  uint64_t* r_full = bars + 2;   // [ST] the rows' factors (32 lanes)
  uint64_t* q_empty = bars + 4;  // [ST] products done
  uint64_t* s_full = bars + 6;   // [2] a step's S^T (buffer = step & 1 = stage)
  uint64_t* s_empty = bars + 8;  // [2] read by 4 warps
  uint64_t* drain = bars + 10;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 11);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_sum = reinterpret_cast<float*>(smem + Cfg::SUM_OFF);

  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bh = blockIdx.y;
  const int b = bh / c.H, h = bh - b * c.H;
  const int len = kv8_len(c, b);
  const int count = kv8_count(counts, b, T);
  const int end = min(kv8_end(c, len, count), max_len);
  const int key0 = blockIdx.x * Cfg::BK;
  if (key0 >= end) return;
  const bool causal = (flags & KF_KV8_CAUSAL) != 0;
  const int rows = min(w.rows, count * G);
  const int first = causal && key0 > len ? (key0 - len) * G : 0;  // first row that sees key0
  const int r_begin = first / BR;
  const int n_steps = (rows + BR - 1) / BR - r_begin;
  if (n_steps <= 0) return;

  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&r_full[s], 32);
      mbar_init(&q_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  // K of the CTA's keys, once.
  if (warp < 8) {
    constexpr int RC = DH / 16;
#pragma unroll
    for (int i = 0; i < (Cfg::LOADS > 0 ? Cfg::LOADS : 1); ++i) {
      const int id = i * 256 + tid;
      if (id >= Cfg::BK * RC) break;
      const int key = key0 + id / RC;
      uint4 r = make_uint4(0u, 0u, 0u, 0u);
      if (key < end) {
        const int page = kv8_page(c, b, key >> c.p_shift);
        if (page >= 0)
          r = __ldg(reinterpret_cast<const uint4*>(
                        c.k + ((static_cast<int64_t>(page) * c.H + h) * c.P + (key & (c.P - 1))) * DH) +
                    id % RC);
      }
      kv8_put16(sK, Cfg::BK, id / RC, id % RC, r, c.fmt);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();

  if (warp == 9) {
    // -------------------------------------------------- rows: Q by TMA, factors
    int issued = 0;
    for (int j = 0; j < n_steps; ++j) {
      const int st = j & 1;
      const uint32_t eph = ((j >> 1) & 1) ^ 1;
      if (j >= 2 && (!mbar_wait(&q_empty[st], eph, abort_flag, KF_DEV_WAIT_TIMEOUT_TMA) ||
                     !mbar_wait(&s_empty[st], eph, abort_flag, KF_DEV_WAIT_TIMEOUT_TMA)))
        break;
      const int row0 = (r_begin + j) * BR;
      if (lane == 0) {
        mbar_arrive_expect_tx(&q_full[st], Cfg::Q_STAGE);
        for (int pl = 0; pl < PL; ++pl)
          for (int ch = 0; ch < Cfg::CH; ++ch)
            tma_load_3d(sQ + st * Cfg::Q_STAGE + pl * Cfg::Q_PLANE + ch * BR * 128, &tmQ,
                        &q_full[st], ch * 64, row0, pl * c.B * c.H + bh);
      }
      ++issued;
      for (int i = lane; i < BR; i += 32) {
        const int row = row0 + i;
        float f = 0.f, nl = -INFINITY;   // rows past the end and empty ones weigh nothing
        if (row < rows) {
          const int64_t at = static_cast<int64_t>(bh) * w.rows + row;
          const float l = __ldg(w.lse + at);
          f = __ldg(w.qf + at);
          nl = l == -INFINITY ? -INFINITY : -l;
        }
        s_row[st * 2 * BR + i] = f;
        s_row[st * 2 * BR + BR + i] = nl;
      }
      mbar_arrive(&r_full[st]);
    }
    if (lane == 0 && *abort_flag)
      for (int j = issued > 2 ? issued - 2 : 0; j < issued; ++j)
        mbar_wait_drain(&q_full[j & 1], (j >> 1) & 1, KF_DEV_WAIT_TIMEOUT_TMA);
  } else if (warp == 8) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_f16(Cfg::BK, BR, 0);
      const uint32_t sKa = smem_u32(sK), sQa = smem_u32(sQ);
      for (int j = 0; j < n_steps; ++j) {
        const int st = j & 1;
        const uint32_t ph = (j >> 1) & 1;
        if (!mbar_wait(&q_full[st], ph, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA)) break;
        if (j >= 2 && !mbar_wait(&s_empty[st], ph ^ 1, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA)) break;
        tc_fence_after();
#pragma unroll
        for (int pl = PL - 1; pl >= 0; --pl)
#pragma unroll
          for (int kk = 0; kk < DH / 16; ++kk) {
            const uint64_t ad = make_smem_desc(sKa + (kk >> 2) * Cfg::BK * 128 + (kk & 3) * 32, 16,
                                               1024, KF_SWIZZLE_128B);
            const uint64_t bd = make_smem_desc(sQa + st * Cfg::Q_STAGE + pl * Cfg::Q_PLANE +
                                                   (kk >> 2) * BR * 128 + (kk & 3) * 32,
                                               16, 1024, KF_SWIZZLE_128B);
            mma_bf16_ss(tmem_base + st * 128, ad, bd, idesc, (pl < PL - 1 || kk > 0) ? 1u : 0u);
          }
        mma_commit(&s_full[st]);
        mma_commit(&q_empty[st]);
      }
      mma_commit(drain);
      mbar_wait_drain(drain, 0, KF_DEV_WAIT_TIMEOUT_MMA);
    }
  } else {
    // -------------------------------------------------- adding: warps 0-3 even steps, 4-7 odd
    const int half = warp >> 2;
    const int quarter = warp & 3;
    const int key = key0 + quarter * 32 + lane;
    int page = -1;
    float ks = 0.f;
    if (key < end) {
      page = kv8_page(c, b, key >> c.p_shift);
      if (page >= 0) ks = __ldg(c.scale + 2 * (static_cast<int64_t>(page) * c.H + h));
    }
    const int see = causal && key > len ? (key - len) * G : 0;  // first row that sees this key
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * 128;
    const uint64_t ks2 = f2_pack(ks, ks);
    float sum = 0.f;
    for (int j = half; j < n_steps; j += 2) {
      const uint32_t ph = (j >> 1) & 1;
      if (!mbar_wait(&r_full[half], ph, abort_flag, KF_DEV_WAIT_TIMEOUT_SOFTMAX) ||
          !mbar_wait(&s_full[half], ph, abort_flag, KF_DEV_WAIT_TIMEOUT_SOFTMAX))
        break;
      tc_fence_after();
      const float* fr = s_row + half * 2 * BR;
      const int skip = see - (r_begin + j) * BR;  // columns below it do not see the key
      const bool mask = __any_sync(0xffffffffu, skip > 0);
      uint64_t acc[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
      for (int cc = 0; cc < BR; cc += 32) {
        float s[32];
        tmem_ld32(t_row + cc, s);
#pragma unroll
        for (int u = 0; u < 32; u += 4) {
          const float4 f = *reinterpret_cast<const float4*>(fr + cc + u);
          const float4 l = *reinterpret_cast<const float4*>(fr + BR + cc + u);
          float e[4];
          f2_unpack(f2_fma(f2_pack(s[u], s[u + 1]), f2_mul(f2_pack(f.x, f.y), ks2),
                           f2_pack(l.x, l.y)), e[0], e[1]);
          f2_unpack(f2_fma(f2_pack(s[u + 2], s[u + 3]), f2_mul(f2_pack(f.z, f.w), ks2),
                           f2_pack(l.z, l.w)), e[2], e[3]);
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            if (mask && cc + u + v < skip) e[v] = -INFINITY;
            e[v] = fast_exp2(e[v]);
          }
          acc[0] = f2_add(acc[0], f2_pack(e[0], e[1]));
          acc[1] = f2_add(acc[1], f2_pack(e[2], e[3]));
        }
      }
      float x0, x1, x2, x3;
      f2_unpack(acc[0], x0, x1);
      f2_unpack(acc[1], x2, x3);
      sum += (x0 + x1) + (x2 + x3);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[half]);
    }
    if (half == 1) s_sum[quarter * 32 + lane] = sum;
    named_bar_sync(1, 256);
    if (half == 0 && page >= 0 && !*abort_flag) {
      float* at = c.weight + (static_cast<int64_t>(page) * c.H + h) * c.P + (key & (c.P - 1));
      *at += sum + s_sum[quarter * 32 + lane];
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) {
    __syncwarp();
    tmem_dealloc(tmem_base, 256);
  }
}

}  // namespace kf
