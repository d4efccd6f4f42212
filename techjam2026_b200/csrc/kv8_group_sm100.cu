// Attention of groups of sequences that share leading pages, on the tcgen05 tensor
// cores: the prompt kernel's pipeline (its roles, TMEM, scales and numbers are
// described there) for rows of several sequences. It differs in where rows come from
// (q is brought in by the softmax warps, without planes in memory), in how work is
// handed out, and in that every CTA leaves parts for the join; the two are kept apart
// because one body for both cost prompts 3 % (chunks over a long cache 390 -> 401 us).
#include "kv8_common.cuh"

namespace kf {

// QP, PP: fp16 planes of q (two for fp32) and of P (two for fp32 and fp16). TILES:
// tiles of 128 query rows. (fp32 at head_dim 128 has room for one: its Q planes fill
// shared memory and its second accumulator TMEM.)
__host__ __device__ constexpr int group_tiles(int dim, int q_planes) {
  return dim == 128 && q_planes == 2 ? 1 : 2;
}
template <int DH, int QP, int PP, int TILES>
struct GroupCfg {
  static constexpr int NT = TILES;
  // Loading warps: 9 to 11, and with one tile 4 to 7, whose rows there are none.
  static constexpr int LW = NT == 1 ? 7 : 3;
  static constexpr int BM = 128;
  static constexpr int BN = 128;                           // keys of a step
  static constexpr int CH = DH > 64 ? 2 : 1;               // 64-column halves of a row
  static constexpr int Q_PLANE = BM * 128 * CH;            // bytes of one tile's plane
  static constexpr int Q_BYTES = NT * QP * Q_PLANE;
  static constexpr int KV_BYTES = BN * 128 * CH;
  static constexpr int ST = 2;                             // stages of K and of V
  static constexpr int RAW = BN * DH;                      // bytes of a tile's codes
  // Raw tiles of K and of V: two where shared memory holds them, so that a copy
  // has a whole step's time.
  static constexpr int RS = DH > 64 && !(NT == 1 && QP == 1) ? 1 : 2;
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

// q of a call with groups, which the softmax warps bring into shared memory.
struct GroupQ {
  const void* q;
  int64_t sb, sh, st;
  int vec;             // 16-byte aligned runs
  float scale_log2;
};

// 32 rows of q, one a lane (at element `base`; < 0: zeros), as one fp16 plane (two)
// in rows r0.. of a tile; returns the lane's factor from the products to log2
// units. A row is taken by as many lanes as it has 16-byte runs of type DT: copied as
// it is to the places of its planes, all rows in flight, then converted there, in a
// loop that is not unrolled. (Code that runs once a CTA costs its fetch, about 200
// clocks for eight instructions: eight runs at a time in registers took 14000 clocks, a
// thread a row as long.)
template <int DH, int DT, int QP, int BM>
__device__ __forceinline__ float group_put_q(const GroupQ& q, int64_t base, uint8_t* tile,
                                              int plane, int r0) {
  constexpr int N = KV8Type<DT>::N, LPR = DH / N, RPI = 32 / LPR;
  const int lane = threadIdx.x & 31, l = lane & (LPR - 1), rr = lane / LPR;
  const int piece = N == 8 ? l : l >> 1;          // of 16 bytes of the plane's row
  auto place = [&](int row) -> uint8_t* {
    return tile + (piece >> 3) * BM * 128 + (r0 + row) * 128 + (((piece & 7) ^ (row & 7)) << 4);
  };
  // fp32: the first run of a piece waits in the first plane, the second in the other
  const int wait_at = N == 4 ? (l & 1) * plane : 0;
#pragma unroll 1
  for (int it = 0; it < LPR; ++it) {
    const int row = it * RPI + rr;
    const int64_t from = __shfl_sync(0xffffffffu, base, row);
    uint8_t* to = place(row) + wait_at;
    if (q.vec) {
      const int64_t at = from < 0 ? 0 : from + l * N;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)),
                   "l"(static_cast<const uint8_t*>(q.q) + at * (DT == KF_DT_F32 ? 4 : 2)),
                   "r"(from < 0 ? 0 : 16)
                   : "memory");
    } else {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (from >= 0) x = KV8Type<DT>::load(q.q, from + l * N, false);
      *reinterpret_cast<uint4*>(to) = x;
    }
  }
  copy_commit();
  copy_wait<0>();
  __syncwarp();
  float mine = 0.f;
#pragma unroll 1
  for (int it = 0; it < LPR; ++it) {
    const int row = it * RPI + rr;
    uint8_t* at = place(row);
    const uint4 x = *reinterpret_cast<const uint4*>(at + wait_at);
    uint32_t m = 0;
    KV8Type<DT>::collect(x, m);
    m = KV8Type<DT>::bits(m);
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    float inv, y[N];
    const float sc = kv8_row_scale(__uint_as_float(m), &inv);
    KV8Type<DT>::values(x, y);
    uint32_t hi[N / 2], lo[N / 2];
#pragma unroll
    for (int v = 0; v < N / 2; ++v) {
      const float a = y[2 * v] * sc, z = y[2 * v + 1] * sc;
      hi[v] = pack_half2(a, z);
      lo[v] = QP == 2 ? pack_half2_rest(a, z, hi[v]) : 0u;
    }
    if constexpr (N == 8) {
      *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[N / 2 - 1]);
    } else {
      __syncwarp();   // (the shuffles before it have all lanes' reads behind them, too)
      at += (l & 1) * 8;
      *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
      if constexpr (QP == 2) *reinterpret_cast<uint2*>(at + plane) = make_uint2(lo[0], lo[1]);
    }
    const float f = __shfl_sync(0xffffffffu, inv, (lane & (RPI - 1)) * LPR);
    if (lane / RPI == it) mine = f;
  }
  return mine * q.scale_log2;
}

// The shared tokens: a CTA an SM takes an equal share of all steps ([group][row tiles][kv
// head][128 keys]), one or more stretches of keys of row tiles; a row tile's
// parts are the CTAs that had some of its steps. (Grids of parts of a fixed size
// ended in a wave of few CTAs: ragged questions on two documents of 8k to 16k
// tokens 234 us for the whole call, this 213.) A step takes 2500 clocks with one tile,
// 4600 with two, 6300 to 7200 at head_dim 128 with two planes of P; a stretch's start and
// end 30000 to 50000, most of it code that is fetched as it first runs. Measured: 64 rows x
// 4 heads against 32k tokens, 8 kv heads of 128, fp16: 85 us.
// OWN: the own tokens; y is the kv head and x [sequence][row tiles][part]. (One body
// that chooses at run time spills more: 226 us for the questions.)
template <int DH, int QP, int PP, int TILES, bool OWN>
__global__ void __launch_bounds__(GroupCfg<DH, QP, PP, TILES>::THREADS, 1)
    kv8_group_kernel(KV8 c, int dtype, const int32_t* __restrict__ counts, int T, int G, int flags,
                     KV8Work w, GroupQ pq, KV8Groups gr) {
  using Cfg = GroupCfg<DH, QP, PP, TILES>;
  constexpr int LW = Cfg::LW;
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
  uint64_t* rk_empty = bars + 24; // [RS] raw codes expanded by the loading warps
  uint64_t* rv_empty = bars + 26; // [RS]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 28);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_vmax = reinterpret_cast<float*>(tmem_slot + 2);  // [12]
  PromptScales* s_sc = reinterpret_cast<PromptScales*>(smem + Cfg::SC_OFF);
  static_assert(sizeof(PromptScales) <= 128, "scale ring");

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto set_up_barriers = [&]() {
    mbar_init(q_full, 4 * NT);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], LW);
      mbar_init(&v_full[s], LW);
      mbar_init(&rk_empty[s], LW);
      mbar_init(&rv_empty[s], LW);
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
  };
  // While the kernel before ends: barriers and TMEM.
  if (tid == 0) set_up_barriers();
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  kv8_begin_of_pair(OWN);   // (every CTA that runs holds its TMEM by now)
  const bool causal = (flags & KF_KV8_CAUSAL) != 0;
  int64_t at = 0, stop = 1, share = 1;   // this CTA's steps of the shared tokens
  int stretch = 0;                       // stretches of keys done
  int4 begin_g = make_int4(0, 0, 0, 0), begin = begin_g;
  if constexpr (!OWN) {
    begin_g = __ldg(gr.record + 2 * blockIdx.x);
    begin = __ldg(gr.record + 2 * blockIdx.x + 1);
    const int64_t all = __ldg(gr.work + gr.N);
    share = __ldg(gr.work + gr.N + 1);
    if (share < 0) share = -share;       // (one stretch a CTA: `all` counts full ones)
    at = blockIdx.x * share;
    stop = min(at + share, all);
  }
  bool more = OWN || at < stop;
  while (more) {
  int b, h, chunk, row0, rows;   // b: whose table row has the pages (the group's first with a new token)
  int end, k0, k1;
  int2 seq = make_int2(0, 0);    // the group's sequences from b on
  bool last_part = false;        // no CTA has later keys of this tile
  if constexpr (!OWN) {
    int4 g = begin_g;
    int item = begin.x, step = begin.y, steps = begin.z;
    chunk = begin.w;
    if (stretch) {
      // The group that holds step `at` of all of them, and its item.
      int lo = 0, hi = gr.N;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(gr.work + mid) <= at)
          lo = mid;
        else
          hi = mid;
      }
      g = __ldg(gr.group + lo);
      steps = (g.x + 127) / 128;
      item = static_cast<int>((at - __ldg(gr.work + lo)) / steps);
      step = 0;
      chunk = 0;
    }
    const int take = static_cast<int>(min(static_cast<int64_t>(steps - step), stop - at));
    h = item % c.H;
    row0 = item / c.H * Cfg::ROWS;
    seq = make_int2(g.z, g.w);
    b = g.z;
    rows = g.y;
    end = g.x;
    k0 = step * BN;
    k1 = min(k0 + take * BN, end);
    last_part = (step + take) * BN >= end;
    at += take;
    more = at < stop;
  } else {
    h = blockIdx.y;
    int i = blockIdx.x;
    const int own = w.chunks - gr.chunks;
    more = false;
    chunk = i % own;
    i /= own;
    b = i / gr.own_tiles;
    row0 = (i - b * gr.own_tiles) * Cfg::ROWS;
    rows = w.rows;
    const int shared = __ldg(gr.of_seq + b);
    const int len = kv8_len(c, b);
    const int count = kv8_count(c, counts, b, T);
    end = kv8_end(c, len, count);
    if (end - shared > gr.max_own) {
      if (tid == 0 && count > 0) record_device_status(KF_DEV_BAD_KV_PAGE);
      end = shared + gr.max_own;
    }
    const int last_row = min(row0 + Cfg::ROWS, rows) - 1;
    const int last_tok = min(last_row / G, count - 1);
    const int reach = last_tok < row0 / G ? 0 : (causal ? min(len + last_tok + 1, end) : end);
    k0 = shared + chunk * w.chunk;
    k1 = min(k0 + w.chunk, reach);
    if (shared == 0 && chunk == 0)
      kv8_no_shared_parts(c, gr, w, b, h, row0, Cfg::ROWS, Cfg::THREADS);
    chunk += gr.chunks;
  }
  // Sequence (from b on) and row within it of a row, and where its numbers are:
  // [B * H][rows of a sequence].
  auto row_of = [&](int row) -> int2 {
    return !OWN ? kv8_group_row(gr, seq, w.rows, G, row) : make_int2(0, row);
  };
  auto spot_of = [&](int2 at) -> int64_t {
    return static_cast<int64_t>((b + at.x) * c.H + h) * w.rows + at.y;
  };
  if (k0 >= k1) {
    // No key: an empty part for the join.
    for (int i = tid; i < Cfg::ROWS; i += Cfg::THREADS) {
      const int row = row0 + i;
      if (row >= rows) break;
      const int64_t spot = spot_of(row_of(row));
      w.ref[spot * w.chunks + chunk] = -INFINITY;
      w.sum[spot * w.chunks + chunk] = 0.f;
    }
    break;
  }
  const int n_steps = (k1 - k0 + BN - 1) / BN;

  float vmax = 0.f;  // the largest V scale of the range
  if (!OWN && stretch) {
    if (tid == 0) set_up_barriers();
    __syncthreads();
  }
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 8) {
    if (lane == 0) {
      // ------------------------------------------------ products
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
    }
  } else if (warp > 8 || (LW == 7 && warp >= 4)) {
    // -------------------------------------------------- loaders (3 or 7 warps)
    // They expand a share of every tile each, without waiting for one
    // another. Warp 9 also copies the raw K tiles, warp 10 the raw V tiles, and
    // warp 11 stages the scales, each half a step after the slot was read.
    int lt = tid - 9 * 32;
    if constexpr (LW == 7) lt += warp < 8 ? 8 * 32 : 0;
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
    if (warp == 9 || warp == 10) {
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
    // The raw slot of step j is asked to hold step j + RS, once all loading warps
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
    {
      // the largest V scale, by the loading warps while the first copies come
      for (int j = (k0 >> c.p_shift) + lt; (j << c.p_shift) < k1; j += 32 * LW) {
        const int page = kv8_page(c, b, j);
        if (page >= 0)
          vmax = fmaxf(vmax, __ldg(c.scale + 2 * (static_cast<int64_t>(page) * c.H + h) + 1));
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, d));
      if (lane == 0) s_vmax[warp] = vmax;
      named_bar_sync(1, 32 * LW);
      if (warp == 11) {
#pragma unroll
        for (int i = 12 - LW - (LW > 3 ? 1 : 0); i < 12; ++i)
          if (i != 8) vmax = fmaxf(vmax, s_vmax[i]);
      }
    }
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
        kv8_expand<DH, KF_KV8_INT8, false, 32 * LW>(rawk + slot * Cfg::RAW, sK + st * Cfg::KV_BYTES, lt, 0, 0);
      else
        kv8_expand<DH, KF_KV8_E4M3, false, 32 * LW>(rawk + slot * Cfg::RAW, sK + st * Cfg::KV_BYTES, lt, 0, 0);
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
            kv8_expand<DH, KF_KV8_INT8, false, 32 * LW>(raw, tile, lt, 0, 0);
          else
            kv8_expand<DH, KF_KV8_INT8, true, 32 * LW>(raw, tile, lt, rows, bad);
        } else {
          if (whole)
            kv8_expand<DH, KF_KV8_E4M3, false, 32 * LW>(raw, tile, lt, 0, 0);
          else
            kv8_expand<DH, KF_KV8_E4M3, true, 32 * LW>(raw, tile, lt, rows, bad);
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
    if ((warp == 9 || warp == 10) && lane == 0) {
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
    int2 my_seq = make_int2(0, row);     // sequence (from b on) and row in it
    bool live = false;                   // the row sees a key
    int limit = 0;
    float qf = 0.f;
    {
      if (row < rows) {
        my_seq = row_of(row);
        live = my_seq.y / G < kv8_count(c, counts, b + my_seq.x, T);
      }
      const int tok = my_seq.y / G;
      // Rows that are not there take all keys of a group like the others (their q is
      // 0): masks cost a third of a step, and nothing of them is written.
      if (!OWN)
        limit = end;
      else if (live)
        limit = causal ? min(kv8_len(c, b) + tok + 1, end) : end;
      const int64_t base = !live ? -1
                                 : (b + my_seq.x) * pq.sb +
                                       static_cast<int64_t>(h * G + my_seq.y - tok * G) * pq.sh +
                                       tok * pq.st;
      uint8_t* tile = sQ + t * QP * Cfg::Q_PLANE;
      if constexpr (QP == 2)
        qf = group_put_q<DH, KF_DT_F32, QP, BM>(pq, base, tile, Cfg::Q_PLANE, quarter * 32);
      else if (dtype == KF_DT_BF16)
        qf = group_put_q<DH, KF_DT_BF16, QP, BM>(pq, base, tile, Cfg::Q_PLANE, quarter * 32);
      else
        qf = group_put_q<DH, KF_DT_F16, QP, BM>(pq, base, tile, Cfg::Q_PLANE, quarter * 32);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    // A warp without a row that sees a key leaves P as it is: no other row reads it.
    const bool idle = !__any_sync(0xffffffffu, live);
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_o = t_lane + Cfg::O_COL + t * Cfg::O_STRIDE;
    const uint32_t t_m = t_lane + Cfg::M_COL + t * Cfg::O_STRIDE;
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
      const uint32_t t_s = t_lane + buf * 128;
      const uint32_t sph = NT == 1 ? (j >> 1) & 1 : j & 1;
      wait(&k_full[st], (j >> 1) & 1);
      wait(&s_full[buf], sph);
      __syncwarp();
      tc_fence_after();
      if (lane == 0 && ok) mbar_arrive(&k_empty[st]);
      if (idle) {
        if (Cfg::SEP && lane == 0 && ok) mbar_arrive(&s_free[t]);
        if (Cfg::SEP && j > 0) wait(&o_done[t], (j - 1) & 1);
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&p_full[buf]);
        continue;
      }
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
        const uint32_t at = Cfg::SEP ? t_lane + Cfg::P_COL + t * 64 + part * 16
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
      if (!live) sum = 0.f, ref = -INFINITY, nan_k = nan_v = false;
#pragma unroll
      for (int i = 12 - LW - (LW > 3 ? 1 : 0); i < 12; ++i)
        if (i != 8) vmax = fmaxf(vmax, s_vmax[i]);
      const int64_t spot = spot_of(my_seq);
      const float nan = __uint_as_float(0x7fc00000u);
      if (nan_k) sum = nan;
      float f = vmax;  // not used where sum is 0
      if (nan_v) f = nan;
      const bool have_m = QP == 2 && n_steps > Cfg::FLUSH;
      // (head_dim 64: rolled, since it runs once a stretch and its code has to be fetched,
      // 216 -> 213 us for questions on two documents; at 128 121 -> 124 for a long one)
#pragma unroll(DH > 64 ? 4 : 1)
      for (int cc = 0; cc < (DH + 31) / 32; ++cc) {
        float o[32];
        tmem_ld32(t_o + cc * 32, o);
        if (have_m) {
          float m[32];
          tmem_ld32(t_m + cc * 32, m);
#pragma unroll
          for (int u = 0; u < 32; ++u) o[u] += m[u];
        }
        constexpr int NC = DH < 32 ? DH : 32;
        // Through this warp's quarter of the tile's Q, which no product reads any
        // more, so that eight lanes write 128 bytes of a row. (A row a lane: 15000
        // clocks for 256 rows of 128.)
        uint8_t* stage = sQ + t * QP * Cfg::Q_PLANE + quarter * 4096;
#pragma unroll
        for (int u = 0; u < 8; ++u)
          *reinterpret_cast<float4*>(stage + lane * 128 + ((u ^ (lane & 7)) << 4)) =
              sum == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                         : make_float4(o[4 * u] * f, o[4 * u + 1] * f, o[4 * u + 2] * f,
                                       o[4 * u + 3] * f);
        __syncwarp();
        const int64_t mine = row < rows && ok ? spot : -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 4 * i + (lane >> 3), piece = lane & 7;
          const int64_t to = __shfl_sync(0xffffffffu, mine, r);
          if (to >= 0 && 4 * piece < NC)
            *reinterpret_cast<float4*>(w.part + (to * w.chunks + chunk) * DH + cc * 32 + 4 * piece) =
                *reinterpret_cast<const float4*>(stage + r * 128 + ((piece ^ (r & 7)) << 4));
        }
        __syncwarp();
      }
      if (row < rows && ok) {
        w.ref[spot * w.chunks + chunk] = ref;
        w.sum[spot * w.chunks + chunk] = sum;
        if (last_part) gr.used[spot] = chunk + 1;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (!more || *abort_flag) break;
  __syncthreads();   // (the flag has been read)
  if (tid == 0)
    for (int i = 0; i < 28; ++i) mbar_inval(bars + i);
  ++stretch;
  }
  if (warp == 8) {
    __syncwarp();
    tmem_dealloc(*tmem_slot, 512);
  }
  kv8_end_of_pair(OWN);
}

}  // namespace kf
