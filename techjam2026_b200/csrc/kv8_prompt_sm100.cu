// Attention of many query rows (prompt chunks) over the 8-bit cache on the
// tcgen05 tensor cores, and the attention weights that such rows give each
// cached token.
//
// kv8_prompt_kernel: one CTA = two tiles of 128 query rows (row = token * G +
// head of the group, so the query heads of a kv head share its K and V) of one
// (sequence, kv head), over a range of keys. Roles:
//   warps 0-3, 4-7  softmax of tile 0 and 1, one thread per row: reads its 128
//                   scores from TMEM, writes P over them as fp16;
//   warp 8          allocates TMEM, loads Q by TMA and issues the products
//                   S = Q K^T (operands in shared memory) and O += P V (P read
//                   from TMEM);
//   warps 9-11      loaders: copy pages of codes to shared memory with bulk
//                   copies a step or two ahead, and expand them to fp16 in
//                   128-byte-swizzled tiles (K: K-major, V: MN-major, the same
//                   bytes: rows are keys); they also stage the scales. (Codes
//                   fetched through registers with a page lookup per piece held
//                   the whole kernel at 6000 clocks a step.)
// TMEM: S0 | S1 (128 columns each), O0 | O1, and P. At head_dim <= 64 with bf16
// q, P has 64 columns of its own per tile, and S(j + 1) is issued as soon as
// step j's scores are in registers, so it is there when their softmax ends.
// Elsewhere P overwrites S and each tile's order is P V(j), then S(j + 1): the
// pipe runs in issue order, so a softmax that sees S(j + 1) knows O holds P V(j)
// and may rescale it at once, and while one tile's products run the other
// tile's softmax has the exponential unit.
// What bounds it: the exponentials, 16 a clock and SM, are 2048 clocks for two
// tiles against 128 keys (the products 1024 at head_dim 64, 2048 at 128). A step
// takes about 3600 clocks at head_dim 64: each softmax warp is busy for 3300 of
// them, 1800 in its exponentials, where 128 scores of 168 registers leave one
// warp little to overlap them with (40 to 80 bytes a thread spill), and about 1000
// in reading the row and its maximum. The schedulers issue in 48 % of the cycles
// there and in 31 % at 128, where P V and S of a tile run between its softmax passes.
// Measured: a chunk of 1024 over 16k tokens, 2 sequences, 16 heads of 64, bf16:
// 274 us for the whole call, 139 GFLOP (505 TFLOP/s); fp16 500, fp32 498: P in the place
// of S, and the second planes' products and conversions between the softmax
// passes. 4 prompts of 2048, 32 heads of 128 on 8 kv heads: bf16 280 us, 138 GFLOP
// (492 TFLOP/s, short rows: 8 steps a CTA), fp16 365, fp32 619 (one tile a CTA).
//
// Numbers as in the split kernel: q rows scaled by powers of two and P relative
// to a lazily moved reference. bf16 q: one fp16 plane of each. fp16 q: two of P
// (P V runs twice; with one, outputs were 1.4 times as far off float64 as fp16's own
// rounding). fp32 q: two of both (both products run twice); page scales enter S exactly and P as the
// ratio to the range's largest V scale.
//
// kv8_prompt_weights_kernel: one CTA = 128 keys against all rows that see
// them: S^T = K Q^T puts a key in each TMEM lane, so a thread adds its key's
// weights in a register over every row, in a fixed order and without atomics.
// Measured: 3 x 4 kv heads of 128, 2800 rows, 3700 tokens, fp32: 115 us, bf16 87.
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

// What the lanes' bounded waits say, for the whole warp: its lanes leave a loop
// together or not at all, since the code after a wait is warp-wide. (The softmax
// warps go without the vote, which cost 10 % at head_dim 64: a lane whose wait has
// failed stays in the loop to its last step, without further waits or arrivals, and
// writes nothing, which costs 1 to 2 %.)
__device__ __forceinline__ bool warp_all(bool ok) { return __all_sync(0xffffffffu, ok); }

// ---------------------------------------------------------------- q planes

// q rows as fp16 planes [QP][B*H][rows][D] and their factors to log2 units. A
// thread holds 16 bytes of each of four rows, neighbours the rest of the row.
// Rows past a sequence's count get zeros. Bound by memory.
constexpr int KV8_PREP_UNROLL = 4;

template <int DT>
__global__ void __launch_bounds__(256)
    kv8_prep_q_kernel(KV8 c, const void* __restrict__ q, int64_t q_sb, int64_t q_sh, int64_t q_st,
                      int vec, const int32_t* __restrict__ counts, int T, int G, float scale_log2,
                      KV8Work w) {
  constexpr int N = KV8Type<DT>::N;
  pdl_launch_dependents();
  pdl_wait();
  const int l_shift = c.d_shift - (N == 8 ? 3 : 2);   // lanes of a row, as a power of two
  const int l = threadIdx.x & ((1 << l_shift) - 1);
  const int rows_of_pass = 256 >> l_shift;
  const int row0 = blockIdx.x * rows_of_pass * KV8_PREP_UNROLL + (threadIdx.x >> l_shift);
  const int bh = blockIdx.y;
  const int b = bh / c.H, h = bh - b * c.H;
  const int real_rows = min(w.rows, kv8_count(c, counts, b, T) * G);
  const int64_t base = b * q_sb + static_cast<int64_t>(h) * G * q_sh;
  uint4 x[KV8_PREP_UNROLL];
#pragma unroll
  for (int i = 0; i < KV8_PREP_UNROLL; ++i) {
    const int row = row0 + i * rows_of_pass;
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (row < real_rows) {
      const int tok = row / G;
      x[i] = KV8Type<DT>::load(q, base + (row - tok * G) * q_sh + tok * q_st + l * N, vec != 0);
    }
  }
  const int64_t plane = static_cast<int64_t>(c.B) * c.H * w.rows * c.D;
#pragma unroll
  for (int i = 0; i < KV8_PREP_UNROLL; ++i) {
    const int row = row0 + i * rows_of_pass;
    uint32_t m = 0;
    KV8Type<DT>::collect(x[i], m);
    m = KV8Type<DT>::bits(m);
    for (int d = 1; d < 1 << l_shift; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (row >= w.rows) continue;
    float inv, y[N];
    const float sc = kv8_row_scale(__uint_as_float(m), &inv);
    KV8Type<DT>::values(x[i], y);
    uint32_t hi[N / 2];
#pragma unroll
    for (int u = 0; u < N; ++u) y[u] *= sc;
#pragma unroll
    for (int u = 0; u < N / 2; ++u) hi[u] = pack_half2(y[2 * u], y[2 * u + 1]);
    uint16_t* at = w.planes + (static_cast<int64_t>(bh) * w.rows + row) * c.D + l * N;
    if constexpr (N == 8) {
      *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[N / 2 - 1]);
    } else {
      *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
      *reinterpret_cast<uint2*>(at + plane) = make_uint2(pack_half2_rest(y[0], y[1], hi[0]),
                                                         pack_half2_rest(y[2], y[3], hi[1]));
    }
    if (l == 0)
      w.qf[static_cast<int64_t>(bh) * w.rows + row] = row < real_rows ? inv * scale_log2 : 0.f;
  }
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

// A tile of 128 rows of raw codes to fp16 in the 128-byte-swizzled layout
// (64-column halves one after the other), by three warps, 16 codes at a time.
// Rows from `rows` on, and groups of 16 rows in `bad`, become zeros (ZERO).
template <int DH, int FMT, bool ZERO>
__device__ __forceinline__ void kv8_expand(const uint8_t* raw, uint8_t* tile, int lt, int rows,
                                           uint32_t bad) {
  constexpr int CW = DH < 64 ? DH : 64;        // columns of a half
  constexpr int RC = CW / 16, RP = 96 / RC;    // pieces of a row of a half, rows of a pass
  constexpr int N = (128 + RP - 1) / RP;
  static_assert(RP % 8 == 0, "swizzle phase");
  const int c16 = lt % RC, r0 = lt / RC;
  const uint32_t ch = static_cast<uint32_t>((c16 * 2) ^ (r0 & 7)) << 4;
  const bool last = r0 + (N - 1) * RP < 128;   // the last pass has rows for some lanes only
#pragma unroll
  for (int x = 0; x < DH / CW; ++x) {
    // Two halves: even rows take half x, odd rows the other one, so that eight
    // lanes touch all banks both when they read and when they write.
    const int half = DH > 64 ? x ^ (r0 & 1) : 0;
    const uint8_t* src = raw + r0 * DH + half * 64 + c16 * 16;
    uint8_t* dst = tile + half * 128 * 128 + r0 * 128;
    uint4 w[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < N - 1 || last) w[i] = *reinterpret_cast<const uint4*>(src + i * RP * DH);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i == N - 1 && !last) break;
      const int r = r0 + i * RP;
      if (ZERO && (r >= rows || ((bad >> (r >> 4)) & 1u))) w[i] = make_uint4(0u, 0u, 0u, 0u);
      uint32_t h[8];
      kv8_cvt4<FMT>(w[i].x, h[0], h[1]);
      kv8_cvt4<FMT>(w[i].y, h[2], h[3]);
      kv8_cvt4<FMT>(w[i].z, h[4], h[5]);
      kv8_cvt4<FMT>(w[i].w, h[6], h[7]);
      *reinterpret_cast<uint4*>(dst + i * RP * 128 + ch) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(dst + i * RP * 128 + (ch ^ 16u)) =
          make_uint4(h[4], h[5], h[6], h[7]);
    }
  }
}

// Untiled copy global -> shared, completion counted on an mbarrier; 16-byte
// aligned addresses and size.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// QP, PP: fp16 planes of q (two for fp32) and of P (two for fp32 and fp16).
template <int DH, int QP, int PP>
struct PromptCfg {
  // Tiles of 128 query rows. fp32 at head_dim 128 takes one: its Q planes fill
  // shared memory and its second accumulator TMEM.
  static constexpr int NT = (DH == 128 && QP == 2) ? 1 : 2;
  static constexpr int BM = 128;
  static constexpr int BN = 128;                           // keys of a step
  static constexpr int CH = DH > 64 ? 2 : 1;               // 64-column halves of a row
  static constexpr int Q_PLANE = BM * 128 * CH;            // bytes of one tile's plane
  static constexpr int Q_BYTES = NT * QP * Q_PLANE;
  static constexpr int KV_BYTES = BN * 128 * CH;
  static constexpr int ST = 2;                             // stages of K and of V
  static constexpr int RAW = BN * DH;                      // bytes of a tile's codes
  static constexpr int RS = DH > 64 ? 1 : 2;               // raw tiles of K and of V
  static constexpr int K_OFF = Q_BYTES;
  static constexpr int V_OFF = K_OFF + ST * KV_BYTES;
  static constexpr int RAWK_OFF = V_OFF + ST * KV_BYTES;
  static constexpr int RAWV_OFF = RAWK_OFF + RS * RAW;
  static constexpr int BAR_OFF = RAWV_OFF + RS * RAW;
  static constexpr int SC_OFF = BAR_OFF + 320;             // page scales of each step
  // Four slots, each read by step j's softmax and rewritten for step j + 4: by
  // then every softmax warp has begun step j + 2.
  static constexpr int SLOTS = 4;
  static constexpr int USED = SC_OFF + SLOTS * 128 + 1024;
  // One CTA per SM (all of TMEM): ask for more than half of shared memory.
  static constexpr int SMEM = USED > 120 * 1024 ? USED : 120 * 1024;
  static constexpr int GROUPS = BN / 16;                   // scale entries of a step
  static constexpr int O_STRIDE = DH < 32 ? 32 : DH;
  static constexpr int O_COL = 256;                        // O of tile t
  // fp32 output: O collects FLUSH steps and is then added to a second
  // accumulator with ordinary fp32 additions. The tensor core's own
  // accumulation drops the bits below the running sum: measured against
  // float64, 2e-9 of relative error per key, 4e-6 after 2048 keys; 5e-7 after 256.
  static constexpr int FLUSH = 2;
  static constexpr int M_COL = O_COL + NT * O_STRIDE;
  // With room in TMEM P has columns of its own, and S of the next step is
  // computed while this step's softmax runs; otherwise P overwrites S.
  static constexpr bool SEP = NT == 2 && PP == 1 && DH <= 64;
  static constexpr int P_COL = O_COL + NT * O_STRIDE;
  static constexpr int ROWS = NT * BM;
  // Twelve warps leave 168 registers a thread: a softmax row's 128 scores and
  // what goes with them.
  static constexpr int THREADS = 12 * 32;
  static_assert(SMEM <= 232448, "smem");
  static_assert((QP == 2 ? M_COL : O_COL) + NT * O_STRIDE <= 512, "TMEM");
  static_assert(!SEP || P_COL + 128 <= 512, "TMEM");
};

// Scales of the keys of one step, by groups of 16 keys.
struct alignas(16) PromptScales {
  float ks[8];
  float ratio[8];     // V scale over the range's largest
  uint32_t bad;       // groups on a refused page
  uint32_t spoiled_k; // groups on a page whose K scale is NaN (its ks is 0 here)
  uint32_t spoiled_v; // the same of V
};

// 128 consecutive columns of this thread's lane, and the wait. The first half's
// registers pass through the last statement, so nothing reads them before it.
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, float (&v)[128]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]), "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]), "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]), "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]), "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
               : "r"(taddr)
               : "memory");
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
               "tcgen05.wait::ld.sync.aligned;"
               : "=f"(v[64]), "=f"(v[65]), "=f"(v[66]), "=f"(v[67]), "=f"(v[68]), "=f"(v[69]), "=f"(v[70]), "=f"(v[71]), "=f"(v[72]), "=f"(v[73]), "=f"(v[74]), "=f"(v[75]), "=f"(v[76]), "=f"(v[77]), "=f"(v[78]), "=f"(v[79]), "=f"(v[80]), "=f"(v[81]), "=f"(v[82]), "=f"(v[83]), "=f"(v[84]), "=f"(v[85]), "=f"(v[86]), "=f"(v[87]), "=f"(v[88]), "=f"(v[89]), "=f"(v[90]), "=f"(v[91]), "=f"(v[92]), "=f"(v[93]), "=f"(v[94]), "=f"(v[95]), "=f"(v[96]), "=f"(v[97]), "=f"(v[98]), "=f"(v[99]), "=f"(v[100]), "=f"(v[101]), "=f"(v[102]), "=f"(v[103]), "=f"(v[104]), "=f"(v[105]), "=f"(v[106]), "=f"(v[107]), "=f"(v[108]), "=f"(v[109]), "=f"(v[110]), "=f"(v[111]), "=f"(v[112]), "=f"(v[113]), "=f"(v[114]), "=f"(v[115]), "=f"(v[116]), "=f"(v[117]), "=f"(v[118]), "=f"(v[119]), "=f"(v[120]), "=f"(v[121]), "=f"(v[122]), "=f"(v[123]), "=f"(v[124]), "=f"(v[125]), "=f"(v[126]), "=f"(v[127])
               : "r"(taddr + 64)
               : "memory");
  asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31]), "+f"(v[32]), "+f"(v[33]), "+f"(v[34]), "+f"(v[35]), "+f"(v[36]), "+f"(v[37]), "+f"(v[38]), "+f"(v[39]), "+f"(v[40]), "+f"(v[41]), "+f"(v[42]), "+f"(v[43]), "+f"(v[44]), "+f"(v[45]), "+f"(v[46]), "+f"(v[47]), "+f"(v[48]), "+f"(v[49]), "+f"(v[50]), "+f"(v[51]), "+f"(v[52]), "+f"(v[53]), "+f"(v[54]), "+f"(v[55]), "+f"(v[56]), "+f"(v[57]), "+f"(v[58]), "+f"(v[59]), "+f"(v[60]), "+f"(v[61]), "+f"(v[62]), "+f"(v[63]) :: "memory");
}
// 16 consecutive columns of this thread's lane, and the wait.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Store 16 consecutive columns (no wait).
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

// Largest of 16 consecutive scores.
__device__ __forceinline__ float max16(const float* s) {
  float m = fmax3(s[0], s[1], s[2]);
  float n = fmax3(s[3], s[4], s[5]);
  m = fmax3(m, s[6], s[7]);
  n = fmax3(n, s[8], s[9]);
  m = fmax3(m, s[10], s[11]);
  n = fmax3(n, s[12], s[13]);
  return fmax3(fmaxf(m, n), s[14], s[15]);
}

template <int DH, int QP, int PP>
__global__ void __launch_bounds__(PromptCfg<DH, QP, PP>::THREADS, 1)
    kv8_prompt_kernel(const __grid_constant__ CUtensorMap tmQ, KV8 c, void* __restrict__ out,
                      int64_t o_sb, int64_t o_sh, int64_t o_st, int dtype, int o_vec,
                      const int32_t* __restrict__ counts, int T, int G, int max_len, int flags,
                      float* __restrict__ lse_out, KV8Work w) {
  using Cfg = PromptCfg<DH, QP, PP>;
  constexpr int BM = Cfg::BM, BN = Cfg::BN, NT = Cfg::NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + Cfg::K_OFF;
  uint8_t* sV = smem + Cfg::V_OFF;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;    // [ST] fp16 tile written, scales staged
  uint64_t* v_full = bars + 3;    // [ST]
  uint64_t* k_empty = bars + 5;   // [ST] S of all tiles done, softmax warps at that step
  uint64_t* v_empty = bars + 7;   // [ST] P V of all tiles done
  uint64_t* s_full = bars + 9;    // [2] by S buffer
  uint64_t* p_full = bars + 11;   // [2] by S buffer, 4 warps
  uint64_t* o_done = bars + 13;   // [2] P V of a step done (not in place: by tile)
  uint64_t* o_final = bars + 15;  // [2]
  uint64_t* drain = bars + 17;
  uint64_t* rk_full = bars + 18;  // [RS] raw codes of K, of V: their bytes
  uint64_t* rv_full = bars + 20;  // [RS]
  uint64_t* s_free = bars + 22;   // [2] S read into registers (P apart), 4 warps
  uint64_t* rk_empty = bars + 24; // [RS] raw codes expanded by the three warps
  uint64_t* rv_empty = bars + 26; // [RS]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 28);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_vmax = reinterpret_cast<float*>(tmem_slot + 2);  // [12]
  PromptScales* s_sc = reinterpret_cast<PromptScales*>(smem + Cfg::SC_OFF);
  static_assert(sizeof(PromptScales) <= 128, "scale ring");

  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bh = blockIdx.z;
  const int b = bh / c.H, h = bh - b * c.H;
  const int chunk = blockIdx.y;
  const int row0 = static_cast<int>(gridDim.x - 1 - blockIdx.x) * Cfg::ROWS;  // heaviest first
  const int len = kv8_len(c, b);
  const int count = kv8_count(c, counts, b, T);
  int end = kv8_end(c, len, count);
  if (end > max_len) {
    if (tid == 0) record_device_status(KF_DEV_BAD_KV_PAGE);
    end = max_len;
  }
  const bool causal = (flags & KF_KV8_CAUSAL) != 0;
  const int last_row = min(row0 + Cfg::ROWS, w.rows) - 1;
  const int last_tok = min(last_row / G, count - 1);
  const int reach = last_tok < row0 / G ? 0 : (causal ? min(len + last_tok + 1, end) : end);
  const int k0 = chunk * w.chunk;
  const int k1 = min(k0 + w.chunk, reach);
  const bool alone = w.chunks == 1;
  if (k0 >= k1) {
    // No key: zeros, or an empty part for the join.
    for (int i = tid; i < Cfg::ROWS; i += Cfg::THREADS) {
      const int row = row0 + i;
      if (row >= w.rows) break;
      const int64_t at = static_cast<int64_t>(bh) * w.rows + row;
      if (!alone) {
        w.ref[at * w.chunks + chunk] = -INFINITY;
        w.sum[at * w.chunks + chunk] = 0.f;
        continue;
      }
      const int tok = row / G, hq = h * G + row - tok * G;
      for (int d = 0; d < DH; ++d)
        kv8_store1(out, b * o_sb + hq * o_sh + tok * o_st + d, dtype, 0.f);
      if (lse_out) lse_out[(static_cast<int64_t>(b) * c.H * G + hq) * T + tok] = -INFINITY;
      if (w.lse) w.lse[at] = -INFINITY;
    }
    return;
  }
  const int n_steps = (k1 - k0 + BN - 1) / BN;

  if (tid == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 3);
      mbar_init(&v_full[s], 3);
      mbar_init(&rk_empty[s], 3);
      mbar_init(&rv_empty[s], 3);
      mbar_init(&rk_full[s], 1);
      mbar_init(&rv_full[s], 1);
      mbar_init(&k_empty[s], 1 + 4 * NT);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&o_final[s], 1);
      mbar_init(&o_done[s], 1);
      mbar_init(&s_free[s], 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // The largest V scale of the range.
  {
    float vmax = 0.f;
    for (int j = (k0 >> c.p_shift) + tid; (j << c.p_shift) < k1; j += Cfg::THREADS) {
      const int page = kv8_page(c, b, j);
      if (page >= 0)
        vmax = fmaxf(vmax, __ldg(c.scale + 2 * (static_cast<int64_t>(page) * c.H + h) + 1));
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
  for (int i = 1; i < 12; ++i) vmax = fmaxf(vmax, s_vmax[i]);

  if (warp == 8) {
    if (lane == 0) {
      // ------------------------------------------------ Q, products
      mbar_arrive_expect_tx(q_full, Cfg::Q_BYTES);
      for (int t = 0; t < NT; ++t)
        for (int pl = 0; pl < QP; ++pl)
          for (int ch = 0; ch < Cfg::CH; ++ch)
            tma_load_3d(sQ + (t * QP + pl) * Cfg::Q_PLANE + ch * BM * 128, &tmQ, q_full, ch * 64,
                        row0 + t * BM, pl * c.B * c.H + bh);
      constexpr uint32_t idesc_s = make_idesc_f16(BM, BN, 0);
      constexpr uint32_t idesc_o = make_idesc_f16(BM, DH, 1);
      const uint32_t sQa = smem_u32(sQ), sKa = smem_u32(sK), sVa = smem_u32(sV);
      // S of tile t and the K tile of `stage` into S buffer `buf`.
      auto issue_s = [&](int t, int buf, int stage) {
#pragma unroll
        for (int pl = QP - 1; pl >= 0; --pl)  // the small plane first
#pragma unroll
          for (int kk = 0; kk < DH / 16; ++kk) {
            const uint64_t ad = make_smem_desc(sQa + (t * QP + pl) * Cfg::Q_PLANE +
                                                   (kk >> 2) * BM * 128 + (kk & 3) * 32,
                                               16, 1024, KF_SWIZZLE_128B);
            const uint64_t bd =
                make_smem_desc(sKa + stage * Cfg::KV_BYTES + (kk >> 2) * BN * 128 + (kk & 3) * 32,
                               16, 1024, KF_SWIZZLE_128B);
            mma_bf16_ss(tmem_base + buf * 128, ad, bd, idesc_s, (pl < QP - 1 || kk > 0) ? 1u : 0u);
          }
        mma_commit(&s_full[buf]);
      };
      // O of tile t += P in S buffer `buf` times the V tile of `stage`.
      auto issue_o = [&](int t, int buf, int stage, bool fresh) {
        const uint32_t p_base = tmem_base + (Cfg::SEP ? Cfg::P_COL + t * 64 : buf * 128);
#pragma unroll
        for (int pl = PP - 1; pl >= 0; --pl)
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk) {
            const uint64_t bd = make_smem_desc(sVa + stage * Cfg::KV_BYTES + kk * 16 * 128, BN * 128,
                                               1024, KF_SWIZZLE_128B);
            mma_f16_ts(tmem_base + Cfg::O_COL + t * Cfg::O_STRIDE,
                       p_base + (Cfg::SEP ? kk * 8 : (kk >> 2) * 64 + pl * 32 + (kk & 3) * 8), bd, idesc_o,
                       (!fresh || pl < PP - 1 || kk > 0) ? 1u : 0u);
          }
      };
      bool ok = mbar_wait(q_full, 0, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA) &&
                mbar_wait(&k_full[0], 0, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < NT; ++t) issue_s(t, t, 0);
        mma_commit(&k_empty[0]);
      }
      if (Cfg::SEP && ok) {
        // Whatever is ready goes next: P V of a tile whose P is written, S of the
        // next step of a tile whose scores are in registers. The last of the two
        // tiles to use a K or V stage releases it.
        int s_next[2] = {1, 1}, p_next[2] = {0, 0};
        long long idle = clock64();
        while (p_next[0] < n_steps || p_next[1] < n_steps) {
          bool progress = false;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int js = s_next[t], jp = p_next[t];
            if (js < n_steps && mbar_test_wait(&s_free[t], (js - 1) & 1) &&
                mbar_test_wait(&k_full[js & 1], (js >> 1) & 1)) {
              tc_fence_after();
              issue_s(t, t, js & 1);
              s_next[t] = js + 1;
              if (s_next[t ^ 1] > js) mma_commit(&k_empty[js & 1]);
              progress = true;
            }
            if (jp < n_steps && mbar_test_wait(&p_full[t], jp & 1) &&
                mbar_test_wait(&v_full[jp & 1], (jp >> 1) & 1)) {
              tc_fence_after();
              issue_o(t, t, jp & 1, jp == 0);
              mma_commit(jp + 1 < n_steps ? &o_done[t] : &o_final[t]);
              p_next[t] = jp + 1;
              if (p_next[t ^ 1] > jp) mma_commit(&v_empty[jp & 1]);
              progress = true;
            }
          }
          if (progress) {
            idle = clock64();
          } else if (*abort_flag) {
            break;
          } else if (clock64() - idle > wait_limit()) {
            *abort_flag = 1;
            record_device_status(KF_DEV_WAIT_TIMEOUT_MMA);
            break;
          }
        }
      }
      for (int j = 0; j < n_steps && ok && !Cfg::SEP; ++j) {
        const int st = j & 1, nx = st ^ 1;
        const uint32_t ph = (j >> 1) & 1, nph = ((j + 1) >> 1) & 1;
        const bool fresh = QP == 2 ? j % Cfg::FLUSH == 0 : j == 0;
        const bool more = j + 1 < n_steps;
        if (NT == 1) {
          // S runs one step ahead of the softmax, in the other buffer: the P
          // there (step j - 1) was consumed by a product issued earlier.
          if (more) {
            ok = mbar_wait(&k_full[nx], nph, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA);
            if (!ok) break;
            tc_fence_after();
            issue_s(0, nx, nx);
            mma_commit(&k_empty[nx]);
          }
          ok = mbar_wait(&v_full[st], ph, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA) &&
               mbar_wait(&p_full[st], ph, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA);
          if (!ok) break;
          tc_fence_after();
          issue_o(0, st, st, fresh);
          mma_commit(more ? o_done : &o_final[0]);
          mma_commit(&v_empty[st]);
        } else {
          ok = mbar_wait(&v_full[st], ph, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA);
          for (int t = 0; t < 2 && ok; ++t) {
            ok = mbar_wait(&p_full[t], j & 1, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA);
            if (!ok) break;
            tc_fence_after();
            issue_o(t, t, st, fresh);
            if (!more) {
              mma_commit(&o_final[t]);
              continue;
            }
            if (t == 0) {
              ok = mbar_wait(&k_full[nx], nph, abort_flag, KF_DEV_WAIT_TIMEOUT_MMA);
              if (!ok) break;
              tc_fence_after();
            }
            issue_s(t, t, nx);
          }
          if (!ok) break;
          mma_commit(&v_empty[st]);
          if (more) mma_commit(&k_empty[nx]);
        }
      }
      mma_commit(drain);
      mbar_wait_drain(drain, 0, KF_DEV_WAIT_TIMEOUT_MMA);
      mbar_wait_drain(q_full, 0, KF_DEV_WAIT_TIMEOUT_MMA);
    }
  } else if (warp > 8) {
    // -------------------------------------------------- loaders (3 warps)
    // The three expand a third of every tile each, without waiting for one
    // another. Warp 9 also copies the raw K tiles, warp 10 the raw V tiles, and
    // warp 11 stages the scales, each half a step after the slot was read.
    const int lt = tid - 9 * 32;
    uint8_t* rawk = smem + Cfg::RAWK_OFF;
    uint8_t* rawv = smem + Cfg::RAWV_OFF;
    const int segs = BN >> c.p_shift;              // pages of a tile (1 to 8)
    const uint32_t seg_bytes = static_cast<uint32_t>(c.P) * DH;
    // Lane g < 8 keeps the pages of group g (16 keys) of the steps ahead: the
    // table entry of step j + RS + 1 is loaded while step j runs, so no copy
    // waits for it. pg[i]: step j + i; -2 no key, -1 the entry is no page.
    int pg[Cfg::RS + 1];
    int entry = -2;
    auto load_entry = [&](int j) {
      const int key = k0 + j * BN + lane * 16;
      entry = -2;
      if (lane < Cfg::GROUPS && key < k1)
        entry = __ldg(c.table + b * c.ld_table + (key >> c.p_shift));
    };
    auto take_entry = [&]() -> int {
      if (entry == -2) return -2;
      if (entry >= 0 && entry < c.pages) return entry;
      record_device_status(KF_DEV_BAD_KV_PAGE);
      return -1;
    };
    // Copies the codes of the pages in lanes 0-7 into a raw slot. A page is
    // copied whole: its slots past the end exist, whatever they hold.
    auto fetch = [&](const uint8_t* pool, uint8_t* raw, uint64_t* full, int page8) {
      const int page = __shfl_sync(0xffffffffu, page8, (lane << (c.p_shift - 4)) & 31);
      const bool live = lane < segs && page >= 0;
      const uint32_t n = __popc(__ballot_sync(0xffffffffu, live));
      if (lane == 0) mbar_arrive_expect_tx(full, n * seg_bytes);
      __syncwarp();
      if (live)
        bulk_load(raw + lane * seg_bytes, pool + (static_cast<int64_t>(page) * c.H + h) * seg_bytes,
                  seg_bytes, full);
    };
#pragma unroll
    for (int i = 0; i <= Cfg::RS; ++i) {
      load_entry(i);
      pg[i] = take_entry();
    }
    load_entry(Cfg::RS + 1);
    int fetched = 0;                               // raw tiles asked for by this warp
    if (warp < 11) {
#pragma unroll
      for (int i = 0; i < Cfg::RS; ++i)
        if (i < n_steps) {
          if (warp == 9)
            fetch(c.k, rawk + i * Cfg::RAW, &rk_full[i], pg[i]);
          else
            fetch(c.v, rawv + i * Cfg::RAW, &rv_full[i], pg[i]);
          ++fetched;
        }
    }
    // The raw slot of step j is asked to hold step j + RS, once all three warps
    // have expanded step j.
    auto refill = [&](const uint8_t* pool, uint8_t* raw, uint64_t* full, uint64_t* empty, int j,
                      int page8) -> bool {
      if (fetched >= n_steps) return true;
      const int slot = j % Cfg::RS;
      if (!warp_all(
              mbar_wait(&empty[slot], (j / Cfg::RS) & 1, abort_flag, KF_DEV_WAIT_TIMEOUT_TMA)))
        return false;
      fetch(pool, raw + slot * Cfg::RAW, &full[slot], page8);
      ++fetched;
      return true;
    };
    // scales of lane g's group: of the current step, loaded one step before
    float2 scale = make_float2(0.f, 0.f);
    auto load_scale = [&](int page8) {
      scale = make_float2(0.f, 0.f);
      if (page8 >= 0)
        scale = __ldg(reinterpret_cast<const float2*>(
            c.scale + 2 * (static_cast<int64_t>(page8) * c.H + h)));
    };
    if (warp == 11) load_scale(pg[0]);
    const float inv_vmax = vmax > 0.f ? 1.f / vmax : 0.f;
    for (int j = 0; j < n_steps; ++j) {
      const int st = j & 1, slot = j % Cfg::RS;
      const uint32_t eph = ((j >> 1) & 1) ^ 1;  // phase of the release two steps back
      const uint32_t rph = (j / Cfg::RS) & 1;
      const uint32_t bad = __ballot_sync(0xffffffffu, lane < Cfg::GROUPS && pg[0] == -1);
      if (!warp_all(mbar_wait(&rk_full[slot], rph, abort_flag, KF_DEV_WAIT_TIMEOUT_TMA) &&
                    (j < 2 || mbar_wait(&k_empty[st], eph, abort_flag, KF_DEV_WAIT_TIMEOUT_TMA))))
        break;
      if (c.fmt == KF_KV8_INT8)
        kv8_expand<DH, KF_KV8_INT8, false>(rawk + slot * Cfg::RAW, sK + st * Cfg::KV_BYTES, lt, 0, 0);
      else
        kv8_expand<DH, KF_KV8_E4M3, false>(rawk + slot * Cfg::RAW, sK + st * Cfg::KV_BYTES, lt, 0, 0);
      fence_proxy_async_smem();
      if (warp == 11) {
        PromptScales& sc = s_sc[j & 3];
        const float sc_k = scale.x, sc_r = scale.y * inv_vmax;
        const uint32_t spoiled_k = __ballot_sync(0xffffffffu, sc_k != sc_k);
        const uint32_t spoiled_v = __ballot_sync(0xffffffffu, sc_r != sc_r);
        if (lane < Cfg::GROUPS) {
          sc.ks[lane] = sc_k == sc_k ? sc_k : 0.f;
          sc.ratio[lane] = sc_r == sc_r ? sc_r : 0.f;
        }
        if (lane == 0) {
          sc.bad = bad;
          sc.spoiled_k = spoiled_k;
          sc.spoiled_v = spoiled_v;
        }
        load_scale(pg[1]);
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&k_full[st]);
        mbar_arrive(&rk_empty[slot]);
      }
      // Refills, where the slot was read half a step ago if there are two, and
      // at once if there is one (its copy then has the rest of the step).
      if (Cfg::RS == 1 && warp == 9 && !refill(c.k, rawk, rk_full, rk_empty, j, pg[Cfg::RS])) break;
      if (Cfg::RS == 2 && warp == 10 && j >= 1 &&
          !refill(c.v, rawv, rv_full, rv_empty, j - 1, pg[Cfg::RS - 1]))
        break;
      if (!warp_all(mbar_wait(&rv_full[slot], rph, abort_flag, KF_DEV_WAIT_TIMEOUT_TMA) &&
                    (j < 2 || mbar_wait(&v_empty[st], eph, abort_flag, KF_DEV_WAIT_TIMEOUT_TMA))))
        break;
      {
        // An e4m3 NaN in a slot past the end must not meet a weight of 0.
        const int rows = k1 - (k0 + j * BN);
        const bool whole = rows >= BN && bad == 0;
        const uint8_t* raw = rawv + slot * Cfg::RAW;
        uint8_t* tile = sV + st * Cfg::KV_BYTES;
        if (c.fmt == KF_KV8_INT8) {
          if (whole)
            kv8_expand<DH, KF_KV8_INT8, false>(raw, tile, lt, 0, 0);
          else
            kv8_expand<DH, KF_KV8_INT8, true>(raw, tile, lt, rows, bad);
        } else {
          if (whole)
            kv8_expand<DH, KF_KV8_E4M3, false>(raw, tile, lt, 0, 0);
          else
            kv8_expand<DH, KF_KV8_E4M3, true>(raw, tile, lt, rows, bad);
        }
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&v_full[st]);
        mbar_arrive(&rv_empty[slot]);
      }
      if (Cfg::RS == 2 && warp == 9 && !refill(c.k, rawk, rk_full, rk_empty, j, pg[Cfg::RS])) break;
      if (Cfg::RS == 1 && warp == 10 && !refill(c.v, rawv, rv_full, rv_empty, j, pg[Cfg::RS])) break;
#pragma unroll
      for (int i = 0; i < Cfg::RS; ++i) pg[i] = pg[i + 1];
      pg[Cfg::RS] = take_entry();
      load_entry(j + Cfg::RS + 2);
    }
    if (warp < 11 && lane == 0) {
      // no copy may be in flight when the CTA leaves
      uint64_t* full = warp == 9 ? rk_full : rv_full;
      for (int j = fetched > Cfg::RS ? fetched - Cfg::RS : 0; j < fetched; ++j)
        mbar_wait_drain(&full[j % Cfg::RS], (j / Cfg::RS) & 1, KF_DEV_WAIT_TIMEOUT_TMA);
    }
  } else if (warp < 4 * NT) {
    // -------------------------------------------------- softmax
    const int t = warp >> 2;
    const int quarter = warp & 3;
    const int row = row0 + t * BM + quarter * 32 + lane;
    const int tok = row / G;
    const int limit = (row < w.rows && tok < count) ? (causal ? min(len + tok + 1, end) : end) : 0;
    const float qf = row < w.rows ? __ldg(w.qf + static_cast<int64_t>(bh) * w.rows + row) : 0.f;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_o = t_row + Cfg::O_COL + t * Cfg::O_STRIDE;
    const uint32_t t_m = t_row + Cfg::M_COL + t * Cfg::O_STRIDE;
    float ref = -INFINITY, sum = 0.f;
    bool ok = true, nan_k = false, nan_v = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (ok) ok = mbar_wait(bar, parity, abort_flag, KF_DEV_WAIT_TIMEOUT_SOFTMAX);
    };
    auto scale_cols = [&](uint32_t at, float alpha) {
#pragma unroll 1
      for (int cc = 0; cc < Cfg::O_STRIDE / 16; ++cc) {
        uint32_t o[16];
        tmem_ld16(at + cc * 16, o);
#pragma unroll
        for (int u = 0; u < 16; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * alpha);
        tmem_st16(at + cc * 16, o);
      }
      tmem_wait_st();
    };
#pragma unroll 1
    for (int j = 0; j < n_steps; ++j) {
      const int st = j & 1;
      const int buf = NT == 1 ? st : t;
      const uint32_t t_s = t_row + buf * 128;
      const uint32_t sph = NT == 1 ? (j >> 1) & 1 : j & 1;
      wait(&k_full[st], (j >> 1) & 1);
      wait(&s_full[buf], sph);
      __syncwarp();
      tc_fence_after();
      if (lane == 0 && ok) mbar_arrive(&k_empty[st]);
      // In place with two tiles, S of this step was issued after P V of the last
      // one, so O is at rest. Otherwise S runs ahead: wait for that product.
      auto at_rest = [&]() {
        if (NT == 2 && !Cfg::SEP) return;
        wait(&o_done[t], (j - 1) & 1);
        __syncwarp();
        tc_fence_after();
      };
      const bool flush = QP == 2 && j > 0 && j % Cfg::FLUSH == 0;
      const bool have_m = QP == 2 && j >= Cfg::FLUSH;  // M holds something
      if (flush) {
        at_rest();
#pragma unroll
        for (int cc = 0; cc < Cfg::O_STRIDE / 16; ++cc) {
          uint32_t o[16], m[16];
          tmem_ld16(t_o + cc * 16, o);
          if (j > Cfg::FLUSH) {
            tmem_ld16(t_m + cc * 16, m);
#pragma unroll
            for (int u = 0; u < 16; ++u)
              o[u] = __float_as_uint(__uint_as_float(o[u]) + __uint_as_float(m[u]));
          }
          tmem_st16(t_m + cc * 16, o);
        }
        tmem_wait_st();
      }
      float s[128];
      tmem_ld128(t_s, s);
      if (Cfg::SEP) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&s_free[t]);
      }
      const PromptScales& sc = s_sc[j & 3];
      const int lim = min(limit, k1) - (k0 + j * BN);
      const uint32_t bad = sc.bad;
      if (__any_sync(0xffffffffu, lim < BN) || bad) {
        uint32_t kw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          kw[i] = ((bad >> (2 * i)) & 1u ? 0u : 0x0000ffffu) |
                  ((bad >> (2 * i + 1)) & 1u ? 0u : 0xffff0000u);
        mask_scores<128>(s, kw, lim);
      }
      if (sc.spoiled_k | sc.spoiled_v) {
        // Rows that see a token of a page whose scale is NaN are NaN: decided
        // per row, since NaN in a product would reach rows that do not.
        if (sc.spoiled_k && lim > 16 * (__ffs(static_cast<int>(sc.spoiled_k)) - 1)) nan_k = true;
        if (sc.spoiled_v && lim > 16 * (__ffs(static_cast<int>(sc.spoiled_v)) - 1)) nan_v = true;
      }
      // A group's factor to log2 units is never 0: a masked score times 0 would
      // be NaN. It is computed where it is used: eight more registers for the
      // factors cost 5 % at head_dim 64 (the row takes 128 of 168). Page scales are
      // positive, so a group's maximum scales with its factor. (The row read twice
      // from TMEM, 32 scores at a time, was 35 % slower.)
      float mx = -INFINITY;
#pragma unroll
      for (int g = 0; g < 8; ++g)
        mx = fmaxf(mx, max16(s + 16 * g) * fmaxf(qf * sc.ks[g], 1e-38f));
      // The reference moves when the maximum has outgrown it by more than the
      // slack.
      float alpha = 1.f;
      const bool move = mx > ref + (KV8_BIAS + KV8_SLACK);
      if (move) {
        if (ref != -INFINITY) alpha = fast_exp2(ref - (mx - KV8_BIAS));
        ref = mx - KV8_BIAS;
        sum *= alpha;
      }
      const bool rescale = j > 0 && __any_sync(0xffffffffu, move);
      if (Cfg::SEP ? j > 0 : rescale) at_rest();  // (P apart: its columns are free then, too)
      if (rescale) {
        if (!flush) scale_cols(t_o, alpha);
        if (have_m) scale_cols(t_m, alpha);
      }
      const float neg = ref == -INFINITY ? 0.f : -ref;
      const uint64_t nr = f2_pack(neg, neg);
      uint64_t acc[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
      for (int part = 0; part < 4; ++part) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const int k = 32 * part + 2 * u;
          const float fg = fmaxf(qf * sc.ks[k >> 4], 1e-38f);
          float x, y;
          f2_unpack(f2_fma(f2_pack(s[k], s[k + 1]), f2_pack(fg, fg), nr), x, y);
          x = fast_exp2(x);
          y = fast_exp2(y);
          acc[u & 1] = f2_add(acc[u & 1], f2_pack(x, y));
          const float r = sc.ratio[k >> 4];
          f2_unpack(f2_mul(f2_pack(x, y), f2_pack(r, r)), x, y);
          hi[u] = pack_half2(x, y);
          if constexpr (PP == 2) lo[u] = pack_half2_rest(x, y, hi[u]);
        }
        const uint32_t at = Cfg::SEP ? t_row + Cfg::P_COL + t * 64 + part * 16
                                     : t_s + (part >> 1) * 64 + (part & 1) * 16;
        tmem_st16(at, hi);
        if constexpr (PP == 2) tmem_st16(at + 32, lo);
      }
      float x0, x1, x2, x3;
      f2_unpack(acc[0], x0, x1);
      f2_unpack(acc[1], x2, x3);
      sum += (x0 + x1) + (x2 + x3);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && ok) mbar_arrive(&p_full[buf]);
    }
    wait(&o_final[t], 0);
    if (__any_sync(0xffffffffu, ok)) {
      tc_fence_after();
      const int64_t at = static_cast<int64_t>(bh) * w.rows + row;
      const int hq = h * G + row - tok * G;
      const float nan = __uint_as_float(0x7fc00000u);
      if (nan_k) sum = nan;
      float f = alone ? vmax / sum : vmax;  // not used where sum is 0
      if (nan_v) f = nan;
      const bool have_m = QP == 2 && n_steps > Cfg::FLUSH;
#pragma unroll
      for (int cc = 0; cc < (DH + 31) / 32; ++cc) {
        float o[32];
        tmem_ld32(t_o + cc * 32, o);
        if (have_m) {
          float m[32];
          tmem_ld32(t_m + cc * 32, m);
#pragma unroll
          for (int u = 0; u < 32; ++u) o[u] += m[u];
        }
        if (row >= w.rows || !ok) continue;
#pragma unroll
        for (int u = 0; u < 32; ++u) o[u] = sum == 0.f ? 0.f : o[u] * f;
        constexpr int NC = DH < 32 ? DH : 32;
        if (alone) {
          kv8_store_run<NC>(out, b * o_sb + hq * o_sh + tok * o_st + cc * 32, dtype, o_vec != 0, o);
        } else {
          float4* p = reinterpret_cast<float4*>(w.part + (at * w.chunks + chunk) * DH + cc * 32);
#pragma unroll
          for (int u = 0; u < NC; u += 4)
            p[u >> 2] = make_float4(o[u], o[u + 1], o[u + 2], o[u + 3]);
        }
      }
      if (row < w.rows && ok) {
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
  if (warp == 8) {
    __syncwarp();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- weights

template <int DH, int QP>
struct WeighCfg {
  static constexpr int BK = 128;                   // keys of a CTA (TMEM lanes)
  static constexpr int BR = 128;                   // query rows of a step
  static constexpr int CH = DH > 64 ? 2 : 1;
  static constexpr int K_BYTES = BK * 128 * CH;
  static constexpr int Q_PLANE = BR * 128 * CH;
  static constexpr int Q_STAGE = QP * Q_PLANE;
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

template <int DH, int QP>
__global__ void __launch_bounds__(WeighCfg<DH, QP>::THREADS)
    kv8_prompt_weights_kernel(const __grid_constant__ CUtensorMap tmQ, KV8 c,
                              const int32_t* __restrict__ counts, int T, int G, int max_len,
                              int flags, KV8Work w) {
  using Cfg = WeighCfg<DH, QP>;
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
  const int count = kv8_count(c, counts, b, T);
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
      if (j >= 2 && !warp_all(mbar_wait(&q_empty[st], eph, abort_flag, KF_DEV_WAIT_TIMEOUT_TMA) &&
                              mbar_wait(&s_empty[st], eph, abort_flag, KF_DEV_WAIT_TIMEOUT_TMA)))
        break;
      const int row0 = (r_begin + j) * BR;
      if (lane == 0) {
        mbar_arrive_expect_tx(&q_full[st], Cfg::Q_STAGE);
        for (int pl = 0; pl < QP; ++pl)
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
    // No copy may be in flight when the CTA leaves, whatever role gives up later.
    if (lane == 0)
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
        for (int pl = QP - 1; pl >= 0; --pl)
#pragma unroll
          for (int kk = 0; kk < DH / 16; ++kk) {
            const uint64_t ad = make_smem_desc(sKa + (kk >> 2) * Cfg::BK * 128 + (kk & 3) * 32, 16,
                                               1024, KF_SWIZZLE_128B);
            const uint64_t bd = make_smem_desc(sQa + st * Cfg::Q_STAGE + pl * Cfg::Q_PLANE +
                                                   (kk >> 2) * BR * 128 + (kk & 3) * 32,
                                               16, 1024, KF_SWIZZLE_128B);
            mma_bf16_ss(tmem_base + st * 128, ad, bd, idesc, (pl < QP - 1 || kk > 0) ? 1u : 0u);
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
      if (!warp_all(mbar_wait(&r_full[half], ph, abort_flag, KF_DEV_WAIT_TIMEOUT_SOFTMAX) &&
                    mbar_wait(&s_full[half], ph, abort_flag, KF_DEV_WAIT_TIMEOUT_SOFTMAX)))
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
