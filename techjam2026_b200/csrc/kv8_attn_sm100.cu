// Attention of a few query rows over the 8-bit cache (single tokens, short
// chunks), split along the keys, and the kernels that join the parts.
//
// What bounds it: the codes. A token of a kv head is 2 * D bytes and serves
// only the G = q_heads / kv_heads query rows of its group, so the arithmetic
// per byte is small and the kernel is a stream over K and V.
//
// One CTA = one chunk of keys of one (sequence, kv head) for a tile of 16 query
// rows (row = token * G + head of the group). Its four warps take the chunk's
// groups of 16 keys in turn, each with its own ring of groups in shared memory,
// filled by asynchronous copies a few groups ahead, and its own running
// reference and sums, joined in shared memory at the end. The lane that feeds a
// code to the tensor core reads it: a contraction may order its terms freely,
// so the lane that holds k-slots {2t, 2t+1, 2t+8, 2t+9} of mma.m16n8k16 owns
// consecutive bytes of a K row (the same ones of q) and consecutive bytes of
// four V rows; the 16-byte pieces of the ring are placed so that those reads
// touch all banks. 16 rows fill the m16 tile; the 128-row tensor-memory
// products would waste 7/8 of theirs here. RH = 1 serves at most 8 rows and
// skips the softmax of the upper half of the tile; a second plane of q or of P
// then takes that half, so one product does both.
// Measured: 16 sequences of 24k tokens, 8 kv heads of 128, four query heads each,
// bf16: 146 us for 787 MB with the join, 5.4 TB/s (0.82 of the copy rate; fp16 151,
// fp32 157); a 65k sequence of 16 heads of 64, fp16: 36 us for 134 MB, 3.7 TB/s, and 6
// to 9 for the join. There the schedulers issue in 65 % of the cycles from 3.5 warps
// each; the stalls after that are fixed latencies and the math pipes, not loads: a
// head width of 64 converts, and pays per 16 keys, as much for half the bytes.
// Rings of 4 slots and 5 or 6 CTAs an
// SM at head_dim 64 were 10 to 25 % slower: the registers they take away cost
// more than their warps hide. (Codes loaded straight into registers, one group
// ahead, left 8 warps an SM and 2.5 TB/s on the first case.)
//
// Numbers. Codes are exact in fp16. A q row is scaled by a power of two to
// [2^14, 2^15) before it becomes one fp16 plane (16-bit q: nothing is lost
// until 2^-28 of the row's largest) or two (fp32 q: 22 bits). P is relative to
// a reference 2^9 below the running maximum, so it uses fp16 up to 2^15 and
// loses precision only below 2^-23 of the largest weight. One plane of P is off
// by 2.0e-4 of the output, which bf16's own rounding (1.65e-3) hides and fp16's
// (2.07e-4) does not: fp16 and fp32 q have two. The V scale of a page is folded into P as the ratio
// to the chunk's largest (<= 1, so P stays in range; what is lost is below 2^-33 of
// the chunk's largest value, whether or not the row sees it). The sum l adds
// the unrounded fp32 weights.
#include "kv8_common.cuh"

namespace kf {

constexpr int KV8_ROWS = 16;            // query rows of a CTA
constexpr int KV8_SPLIT_ROWS = 64;      // query rows of a kv head that this path serves
constexpr int KV8_CHUNK_MAX = 4096;     // keys of a CTA: at most 256 pages of 16
constexpr float KV8_BIAS = 9.f;         // log2 of P's largest value after a rescale
constexpr float KV8_SLACK = 6.f;        // growth of the maximum that needs no rescale

// Layout of the workspace: per (sequence, kv head, padded row, chunk) the
// reference and the sum, then the partial outputs, then (track) the scores.
struct KV8Work {
  float* ref;     // [B*H][rows][chunks]
  float* sum;     // [B*H][rows][chunks]
  float* part;    // [B*H][rows][chunks][D]
  float* lse;     // [B*H][rows]: log2 of the softmax's sum
  float* score;   // [B*H][rows][ld_score] (few rows and track), in log2 units
  uint16_t* planes;  // many rows: q as fp16 planes [QP][B*H][rows][D]
  float* qf;         // and their factors [B*H][rows]
  int64_t ld_score;
  int rows;       // T * G
  int chunks;
  int chunk;      // keys of a chunk
  bool prompt;    // the tensor-memory kernel runs
};

// Groups of sequences that share leading pages (kf_kv8_attention_shared). The
// rows of a call are cut twice: the rows of a whole group against the tokens
// that it shares, and the rows of each sequence against its other tokens.
struct KV8Groups {
  const int32_t* starts;  // [N + 1]: group n is the sequences starts[n] .. starts[n + 1] - 1
  const int32_t* shared;  // [N]: tokens its table rows have in common
  const int32_t* live;    // [B + 1]: new tokens of the sequences before; null: T of each
  int N;
  int max_shared;         // whole pages
  int max_own;
  int tiles;              // row tiles of all groups, at most
  int chunks, chunk;      // parts of the shared tokens; KV8Work has those of the others
  int own_tiles;          // row tiles of a sequence
  // Of kv8_groups_kernel, for the tensor-memory kernel (null otherwise):
  const int4* group;      // [N]: shared tokens, rows, first sequence, one past the last
  const int64_t* work;    // [N + 1]: steps of the groups before; then a CTA's steps
  const int4* record;     // [ctas][2]: where a CTA begins: the group's entry, and {item,
                          // step, steps of an item, part}; item = row tile * H + head
  const int32_t* of_seq;  // [B]: tokens that a sequence shares
  int32_t* used;          // [B * H][rows]: parts of the shared tokens that a row has
  int least;              // steps of a part, at least
};

// The sequences of group n; none (recorded) where starts is out of order.
__device__ __forceinline__ int2 kv8_group(const KV8Groups& gr, int B, int n) {
  const int a = __ldg(gr.starts + n), z = __ldg(gr.starts + n + 1);
  if (a < 0 || z < a || z > B) {
    record_device_status(KF_DEV_BAD_GROUPS);
    return make_int2(0, 0);
  }
  return make_int2(a, z);
}
// Tokens that group n shares (x), of whole pages that all of its sequences with a new
// token hold, and the first such sequence (y), whose table row names the pages. (One
// without a new token reads nothing: its length, 0 or negative in an idle place,
// would leave the others without what they share.) All lanes of a warp call this
// together.
__device__ __forceinline__ int2 kv8_group_tokens(const KV8& c, const KV8Groups& gr,
                                                 const int32_t* counts, int T, int n, int2 seq) {
  int s = __ldg(gr.shared + n);
  s = s < 0 ? 0 : min(s, gr.max_shared);
  int first = INT32_MAX;
  for (int b = seq.x + (threadIdx.x & 31); b < seq.y; b += 32) {
    // (a length beyond the table's reach, which max_shared is within, is recorded by
    // the sequence's own tokens)
    const int len = __ldg(c.lens + b), count = counts ? __ldg(counts + b) : T;
    if (len >= 0 && count > 0) {
      s = min(s, len);
      first = min(first, b);
    }
  }
  s = __reduce_min_sync(0xffffffffu, s);
  first = __reduce_min_sync(0xffffffffu, first);
  if (first == INT32_MAX) return make_int2(0, seq.x);
  return make_int2(s & ~(c.P - 1), first);
}
// Query rows of a group's sequences: the rows of their new tokens one after
// another, or where `live` is null `per` rows of each (with tokens past counts).
__device__ __forceinline__ int kv8_group_rows(const KV8Groups& gr, int2 seq, int per, int G) {
  return gr.live ? (__ldg(gr.live + seq.y) - __ldg(gr.live + seq.x)) * G : (seq.y - seq.x) * per;
}
// Sequence (x, counted from the group's first) and row within it (y) of a row.
__device__ __forceinline__ int2 kv8_group_row(const KV8Groups& gr, int2 seq, int per, int G,
                                              int row) {
  if (!gr.live) {
    const int m = row / per;
    return make_int2(m, row - m * per);
  }
  const int first = __ldg(gr.live + seq.x), tok = row / G;
  int lo = seq.x, hi = seq.y;       // the last sequence that begins at or before tok
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(gr.live + mid) - first <= tok)
      lo = mid;
    else
      hi = mid;
  }
  return make_int2(lo - seq.x, row - (__ldg(gr.live + lo) - first) * G);
}
// Group and tile of the index-th tile of `tile` rows; n < 0: there are fewer. All
// lanes of a warp call this together.
struct KV8GroupTile {
  int n, tile, rows;
  int2 seq;
};
__device__ __forceinline__ KV8GroupTile kv8_group_tile(const KV8Groups& gr, int B, int per, int G,
                                                       int tile, int index) {
  const int lane = threadIdx.x & 31;
  for (int base = 0; base < gr.N; base += 32) {
    const int2 seq = base + lane < gr.N ? kv8_group(gr, B, base + lane) : make_int2(0, 0);
    const int rows = kv8_group_rows(gr, seq, per, G);
    const int tiles = (rows + tile - 1) / tile;
    int sum = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, sum > index);
    if (past) {
      const int l = __ffs(static_cast<int>(past)) - 1;
      KV8GroupTile t;
      t.n = base + l;
      t.tile = index - __shfl_sync(0xffffffffu, sum - tiles, l);
      t.rows = __shfl_sync(0xffffffffu, rows, l);
      t.seq.x = __shfl_sync(0xffffffffu, seq.x, l);
      t.seq.y = __shfl_sync(0xffffffffu, seq.y, l);
      return t;
    }
    index -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return KV8GroupTile{-1, 0, 0, make_int2(0, 0)};
}
// Tokens that sequence b shares with its group (0: it is in none).
__device__ __forceinline__ int kv8_shared_of(const KV8& c, const KV8Groups& gr,
                                             const int32_t* counts, int T, int b) {
  if (gr.of_seq) return __ldg(gr.of_seq + b);
  const int lane = threadIdx.x & 31;
  for (int base = 0; base < gr.N; base += 32) {
    const int2 seq = base + lane < gr.N ? kv8_group(gr, c.B, base + lane) : make_int2(0, 0);
    const uint32_t in = __ballot_sync(0xffffffffu, b >= seq.x && b < seq.y);
    if (in) {
      const int l = __ffs(static_cast<int>(in)) - 1;
      return kv8_group_tokens(c, gr, counts, T, base + l,
                              make_int2(__shfl_sync(0xffffffffu, seq.x, l),
                                        __shfl_sync(0xffffffffu, seq.y, l))).x;
    }
  }
  return 0;
}

// The kernel of the own tokens (gr.tiles = 0) runs beside that of the shared ones: it
// begins without waiting for it, and ends after it, so that the join has to wait for
// one kernel. What it reads besides is complete by then: the shared kernel's CTAs
// signal only after their own wait, when all that ran before (the groups' lists, q,
// the cache) has ended and is visible to them, and the own kernel's CTAs start after
// all of those signals. A grid is promised to see such writes at its wait only, so
// each of its threads begins with a fence at the GPU's scope, which leaves nothing
// older in its SM's L1 cache for its reads, and not with a wait, which
// would run the two kernels one after the other (64 samples 30.6 -> 36.4 us, uneven
// groups 94 -> 100, questions 222 -> 234; the fence costs 0.3 us of the 64 samples' 31,
// and nothing that shows elsewhere).
__device__ __forceinline__ void kv8_begin_of_pair(bool own) {
  if (own)
    __threadfence();
  else
    pdl_wait();
  pdl_launch_dependents();   // (only now: see above)
}
__device__ __forceinline__ void kv8_end_of_pair(bool own) {
  if (own) pdl_wait();
}
// Empty parts in the places of the shared tokens, or none, for rows that share
// nothing.
__device__ __forceinline__ void kv8_no_shared_parts(const KV8& c, const KV8Groups& gr,
                                                    const KV8Work& w, int b, int h, int row0,
                                                    int tile, int threads) {
  if (gr.used) {
    for (int u = threadIdx.x; u < tile && row0 + u < w.rows; u += threads)
      gr.used[static_cast<int64_t>(b * c.H + h) * w.rows + row0 + u] = 0;
    return;
  }
  for (int u = threadIdx.x; u < tile * gr.chunks; u += threads) {
    const int row = row0 + u / gr.chunks;
    if (row >= w.rows) break;
    const int64_t at =
        (static_cast<int64_t>(b * c.H + h) * w.rows + row) * w.chunks + u % gr.chunks;
    w.ref[at] = -INFINITY;
    w.sum[at] = 0.f;
  }
}

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The product alone, without an earlier accumulator.
__device__ __forceinline__ void mma_f16_16816_first(float (&d)[4], uint32_t a0, uint32_t a1,
                                                    uint32_t a2, uint32_t a3, uint32_t b0,
                                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

template <int BYTES>
__device__ __forceinline__ void read_bytes(const uint8_t* p, uint32_t* w) {
  if constexpr (BYTES == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else if constexpr (BYTES == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
}

__device__ __forceinline__ void copy16_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The rest of a and b after pack_half2, as a second fp16 plane.
__device__ __forceinline__ uint32_t pack_half2_rest(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return pack_half2(a - f.x, b - f.y);
}

// Power of two that brings a row whose largest magnitude is `amax` to
// [2^14, 2^15), as a biased exponent pattern; 1 for a row of zeros or one that
// holds an infinity or a NaN.
__device__ __forceinline__ float kv8_row_scale(float amax, float* inverse) {
  const uint32_t ex = __float_as_uint(amax) >> 23;
  if (amax == 0.f || ex == 255u) {
    *inverse = 1.f;
    return 1.f;
  }
  const int e = min(max(268 - static_cast<int>(ex), 1), 253);
  *inverse = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
  return __uint_as_float(static_cast<uint32_t>(e) << 23);
}

// The q fragments of 16 rows: lane (g, t) holds rows g and g + 8, the K bytes
// it owns (see above). qf[r]: factor from the products to log2 units.
template <int DH, int QP, int RH>
struct QFrag {
  static constexpr int EPT = DH / 4 < 16 ? DH / 4 : 16;  // consecutive elements of a piece
  static constexpr int NPC = DH / 4 / EPT;               // pieces (64 elements apart)
  static constexpr int KS = DH / 16;                     // k-steps
  // RH = 1: rows g + 8 are zeros, or with two planes the second plane.
  static constexpr int NP = RH == 1 ? 1 : QP;            // products per k-step
  uint32_t a[NP][KS][4];
  float qf[RH];

  // at(row): the element where a row of q begins.
  template <class At>
  __device__ __forceinline__ void load(const void* q, At&& at, int dtype, bool vec, int row0,
                                       int rows, float scale_log2) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if constexpr (RH == 1 && QP == 1) {
#pragma unroll
      for (int s = 0; s < KS; ++s) a[0][s][1] = a[0][s][3] = 0u;
    }
#pragma unroll
    for (int r = 0; r < RH; ++r) {
      const int row = row0 + g + 8 * r;
      float x[NPC * EPT];
      float amax = 0.f;
      if (row < rows) {
        const int64_t base = at(row);
#pragma unroll
        for (int p = 0; p < NPC; ++p)
#pragma unroll
          for (int e = 0; e < EPT; e += 4) {
            float y[4];
            kv8_load4(q, base + p * 64 + t * EPT + e, dtype, vec, y);
#pragma unroll
            for (int u = 0; u < 4; ++u) x[p * EPT + e + u] = y[u];
          }
      } else {
#pragma unroll
        for (int e = 0; e < NPC * EPT; ++e) x[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < NPC * EPT; ++e)
        amax = __uint_as_float(max(__float_as_uint(amax), __float_as_uint(fabsf(x[e]))));
#pragma unroll
      for (int d = 1; d <= 2; d <<= 1)
        amax = __uint_as_float(
            max(__float_as_uint(amax), __shfl_xor_sync(0xffffffffu, __float_as_uint(amax), d)));
      float inv;
      const float sc = kv8_row_scale(amax, &inv);
      qf[r] = inv * scale_log2;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        float y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) y[u] = x[4 * s + u] * sc;
        a[0][s][r] = pack_half2(y[0], y[1]);
        a[0][s][2 + r] = pack_half2(y[2], y[3]);
        if constexpr (QP == 2) {
          a[NP - 1][s][RH == 1 ? 1 : r] = pack_half2_rest(y[0], y[1], a[0][s][r]);
          a[NP - 1][s][RH == 1 ? 3 : 2 + r] = pack_half2_rest(y[2], y[3], a[0][s][2 + r]);
        }
      }
    }
  }
};

// A ring slot holds 16 keys: K rows, then V rows, as 16-byte pieces. Piece
// `p` (row-major over 16 rows of DH bytes) goes to these places, so that the
// eight lanes (16-byte reads) or sixteen (8-byte) of a read's phase fall on
// different banks: K, 128-byte rows: odd rows swap their halves; V, 128-byte
// rows: pieces are xored with row & 7 (a read takes rows 0, 2, 4, 6), 64-byte
// rows: with twice the number of the 128-byte line.
template <int DH>
__device__ __forceinline__ int k_place(int p) {
  if constexpr (DH == 128) return p ^ (((p >> 3) & 1) << 2);
  return p;
}
template <int DH>
__device__ __forceinline__ int v_place(int p) {
  if constexpr (DH == 128) return p ^ ((p >> 3) & 7);
  if constexpr (DH == 64) return p ^ (((p >> 3) & 3) << 1);
  return p;
}

// Codes of K for 16 keys as one lane owns them: two n8 tiles of keys.
template <int DH>
struct KBytes {
  static constexpr int EPT = DH / 4 < 16 ? DH / 4 : 16;
  static constexpr int NPC = DH / 4 / EPT;
  uint32_t w[2][DH / 16];
  __device__ __forceinline__ void read(const uint8_t* slot) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int p = 0; p < NPC; ++p) {
        const int at = (8 * n + g) * DH + p * 64 + t * EPT;  // byte
        read_bytes<EPT>(slot + k_place<DH>(at >> 4) * 16 + (at & 15), &w[n][p * (EPT / 4)]);
      }
  }
};
template <int DH>
struct VBytes {
  static constexpr int VB = DH / 8;            // consecutive bytes of a row
  static constexpr int W = VB < 4 ? 1 : VB / 4;
  uint32_t w[4][W];                            // keys 2t, 2t+1, 8+2t, 9+2t
  __device__ __forceinline__ void read(const uint8_t* slot) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = ((i >> 1) * 8 + 2 * t + (i & 1)) * DH + g * VB;
      read_bytes<VB>(slot + 16 * DH + v_place<DH>(at >> 4) * 16 + (at & 15), w[i]);
    }
  }
};

template <int DH>
struct SplitCfg {
  static constexpr int SLOT = 32 * DH;              // bytes of 16 keys, K and V
  static constexpr int DEPTH = DH == 128 ? 4 : 6;   // slots of a warp's ring
  static constexpr int RING = 4 * DEPTH * SLOT;
  static constexpr int JOIN = 4 * KV8_ROWS * DH * 4;
  static constexpr int SMEM = RING > JOIN ? RING : JOIN;
  // CTAs an SM is to hold: what the rings (and, at 128, the registers) allow.
  static constexpr int min_blocks(int q_planes) { return DH == 128 ? (q_planes == 1 ? 3 : 2) : 4; }
};

// Products of 16 q rows with 16 keys: d[n][.] in the m16n8 accumulator layout.
template <int DH, int FMT, int QP, int RH>
__device__ __forceinline__ void score_tile(const QFrag<DH, QP, RH>& q, const KBytes<DH>& kb,
                                           float (&d)[2][4]) {
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
#pragma unroll
    for (int s = 0; s < DH / 16; ++s) {
      uint32_t b0, b1;
      kv8_cvt4<FMT>(kb.w[n][s], b0, b1);
      if constexpr (QP == 2 && RH == 2)
        mma_f16_16816(d[n], q.a[1][s][0], q.a[1][s][1], q.a[1][s][2], q.a[1][s][3], b0, b1);
      mma_f16_16816(d[n], q.a[0][s][0], q.a[0][s][1], q.a[0][s][2], q.a[0][s][3], b0, b1);
    }
    if constexpr (QP == 2 && RH == 1) {
      d[n][0] += d[n][2];
      d[n][1] += d[n][3];
    }
  }
}

template <class T>
__device__ __forceinline__ const T& kv8_the(const T& one) {
  return one;
}

// QP, PP: fp16 planes of q and of P. SH: the call has groups, one KV8Groups (a pack, since
// a parameter that plain calls do not need costs each 0.3 us of host); y is then the kv
// head, and the CTAs (x) are [row tile of a group][part of its shared tokens] (none if
// its tiles are 0), then [sequence][row tile][part of its own tokens].
template <int DH, int FMT, int QP, int PP, int RH, class... Groups>
__global__ void __launch_bounds__(128, SplitCfg<DH>::min_blocks(QP))
    kv8_split_kernel(KV8 c, const void* __restrict__ q, int64_t q_sb, int64_t q_sh, int64_t q_st,
                     void* __restrict__ out, int64_t o_sb, int64_t o_sh, int64_t o_st, int dtype,
                     int vec, const int32_t* __restrict__ counts, int T, int G, int max_len,
                     float scale_log2, int flags, float* __restrict__ lse_out, KV8Work w,
                     Groups... groups) {
  constexpr bool SH = sizeof...(Groups) > 0;
  constexpr int NT = DH / 8;  // n8 tiles of the output
  __shared__ int s_page[KV8_CHUNK_MAX / 16];
  __shared__ float s_ks[KV8_CHUNK_MAX / 16];
  __shared__ float s_vs[KV8_CHUNK_MAX / 16];
  __shared__ float s_vmax[4];
  extern __shared__ __align__(128) uint8_t s_ring[];
  __shared__ float s_ref[4][KV8_ROWS], s_sum[4][KV8_ROWS];
  __shared__ int2 s_row[SH ? KV8_ROWS : 1];
  if constexpr (!SH) {
    pdl_launch_dependents();
    pdl_wait();
  } else {
    kv8_begin_of_pair(kv8_the(groups...).tiles == 0);
  }
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const bool causal = (flags & KF_KV8_CAUSAL) != 0;
  int chunk, row0, h, b;    // b: the sequence, or the group's first one
  int pages_of;             // whose table row has the pages
  int rows;                 // rows that the tile is cut from
  int end;                  // no key is at or past it
  int limit[RH];            // the rows' own limits
  int k0, k1;               // the CTA's keys
  if constexpr (!SH) {
    chunk = blockIdx.x;
    row0 = blockIdx.y * KV8_ROWS;
    const int bh = blockIdx.z;
    b = bh / c.H;
    h = bh - b * c.H;
    pages_of = b;
    rows = w.rows;
    const int len = kv8_len(c, b);
    const int count = kv8_count(c, counts, b, T);
    end = kv8_end(c, len, count);
    if (end > max_len) {
      if (tid == 0) record_device_status(KF_DEV_BAD_KV_PAGE);
      end = max_len;
    }
    // Last key that any row of this tile sees.
    int reach = 0;
#pragma unroll
    for (int r = 0; r < RH; ++r) {
      const int row = row0 + g + 8 * r;
      const int tok = row / G;
      limit[r] = (row < w.rows && tok < count) ? (causal ? min(len + tok + 1, end) : end) : 0;
    }
    {
      const int last_row = min(row0 + KV8_ROWS, w.rows) - 1;
      const int last_tok = min(last_row / G, count - 1);
      reach = last_tok < row0 / G ? 0 : (causal ? min(len + last_tok + 1, end) : end);
    }
    k0 = chunk * w.chunk;
    k1 = min(k0 + w.chunk, reach);
  } else {
    const KV8Groups& gr = kv8_the(groups...);
    h = blockIdx.y;
    int i = blockIdx.x;
    if (i < gr.tiles * gr.chunks) {
      chunk = i % gr.chunks;
      const KV8GroupTile tl = kv8_group_tile(gr, c.B, w.rows, G, KV8_ROWS, i / gr.chunks);
      if (tl.n < 0) return;
      b = tl.seq.x;
      row0 = tl.tile * KV8_ROWS;
      rows = tl.rows;
      // every row of a sequence that takes its token sees all that is shared
      const int2 common = kv8_group_tokens(c, gr, counts, T, tl.n, tl.seq);
      end = common.x;
      pages_of = common.y;
      k0 = chunk * gr.chunk;
      k1 = min(k0 + gr.chunk, end);
      if (end == 0) return;  // the sequences' own CTAs leave the empty parts
      if (tid < KV8_ROWS && row0 + tid < rows)
        s_row[tid] = kv8_group_row(gr, tl.seq, w.rows, G, row0 + tid);
      __syncthreads();
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        limit[r] = 0;
        if (row0 + g + 8 * r < rows) {
          const int2 at = s_row[g + 8 * r];
          if (at.y / G < kv8_count(c, counts, b + at.x, T)) limit[r] = end;
        }
      }
    } else {
      i -= gr.tiles * gr.chunks;
      const int own = w.chunks - gr.chunks;
      chunk = i % own;
      i /= own;
      b = i / gr.own_tiles;
      pages_of = b;
      row0 = (i - b * gr.own_tiles) * KV8_ROWS;
      rows = w.rows;
      const int shared = kv8_shared_of(c, gr, counts, T, b);
      const int len = kv8_len(c, b);
      const int count = kv8_count(c, counts, b, T);
      end = kv8_end(c, len, count);
      if (end - shared > gr.max_own) {
        if (tid == 0 && count > 0) record_device_status(KF_DEV_BAD_KV_PAGE);
        end = shared + gr.max_own;
      }
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        const int row = row0 + g + 8 * r;
        const int tok = row / G;
        limit[r] = (row < rows && tok < count) ? (causal ? min(len + tok + 1, end) : end) : 0;
      }
      if (tid < KV8_ROWS) s_row[tid] = make_int2(0, row0 + tid);
      __syncthreads();
      const int last_row = min(row0 + KV8_ROWS, rows) - 1;
      const int last_tok = min(last_row / G, count - 1);
      const int reach = last_tok < row0 / G ? 0 : (causal ? min(len + last_tok + 1, end) : end);
      k0 = shared + chunk * w.chunk;
      k1 = min(k0 + w.chunk, reach);
      if (shared == 0 && chunk == 0) kv8_no_shared_parts(c, gr, w, b, h, row0, KV8_ROWS, 128);
      chunk += gr.chunks;
    }
  }
  // Where a row's numbers are: [B * H][rows of a sequence]. The row comes in parts, each
  // added in 64 bits: with sums in 32 the compiler holds other values, and a token of 64
  // ragged sequences with the record takes 43.1 us instead of 42.5.
  auto spot = [&](auto... row) -> int64_t {
    if constexpr (!SH) return (static_cast<int64_t>(blockIdx.z) * w.rows + ... + row);
    const int2 at = s_row[SH ? (row + ...) - row0 : 0];
    return static_cast<int64_t>((b + at.x) * c.H + h) * w.rows + at.y;
  };
  const bool alone = w.chunks == 1;
  if (k0 >= k1 && !alone) {
    // nothing here: the join reads this chunk's sums all the same
    for (int r = tid; r < KV8_ROWS; r += 128)
      if (row0 + r < rows) {
        const int64_t at = spot(row0, r) * w.chunks + chunk;
        w.ref[at] = -INFINITY;
        w.sum[at] = 0.f;
      }
    if constexpr (SH) kv8_end_of_pair(kv8_the(groups...).tiles == 0);
    return;
  }
  const int j0 = k0 >> c.p_shift;
  float vmax = 0.f;
  for (int j = j0 + tid; (j << c.p_shift) < k1; j += 128) {
    const int page = kv8_page(c, pages_of, j);
    s_page[j - j0] = page;
    float2 s = make_float2(0.f, 0.f);
    if (page >= 0) s = *reinterpret_cast<const float2*>(c.scale + 2 * (static_cast<int64_t>(page) * c.H + h));
    s_ks[j - j0] = s.x;
    s_vs[j - j0] = s.y;
    vmax = fmaxf(vmax, s.y);
  }
  QFrag<DH, QP, RH> qa;
  qa.load(q, [&](int row) {
    int m = 0;
    if constexpr (SH) {
      const int2 at = s_row[row - row0];
      m = at.x;
      row = at.y;
    }
    const int tok = row / G;
    return (b + m) * q_sb + static_cast<int64_t>(h * G + row - tok * G) * q_sh + tok * q_st;
  }, dtype, vec != 0, row0, rows, scale_log2);
#pragma unroll
  for (int d = 16; d; d >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, d));
  if (lane == 0) s_vmax[warp] = vmax;
  __syncthreads();
  vmax = fmaxf(fmaxf(s_vmax[0], s_vmax[1]), fmaxf(s_vmax[2], s_vmax[3]));
  const float inv_vmax = vmax > 0.f ? 1.f / vmax : 0.f;

  // With two planes of P, O collects the products of 16 keys by fp32 additions: the
  // tensor core's own accumulation drops what lies below the running sum (with
  // 1024 keys a warp 1.4e-6 to 2.9e-6 against float64; so 4e-7 to 8e-7, in the
  // same time).
  constexpr int OW = PP == 2 ? 2 * RH : 4;  // of a tile's columns, held by a lane
  float o[NT][OW];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < OW; ++e) o[n][e] = 0.f;
  float ref[RH], sum[RH];
#pragma unroll
  for (int r = 0; r < RH; ++r) {
    ref[r] = -INFINITY;
    sum[r] = 0.f;
  }

  // The warp's ring: group i of this warp is keys k0 + 64 i + 16 warp and up.
  using Cfg = SplitCfg<DH>;
  uint8_t* ring = s_ring + warp * Cfg::DEPTH * Cfg::SLOT;
  const int page_bytes = c.P * DH;
  auto fetch = [&](int key, int slot) {
    if (key < k1) {
      const int page = s_page[(key >> c.p_shift) - j0];
      const int64_t at = (static_cast<int64_t>(page < 0 ? 0 : page) * c.H + h) * page_bytes +
                         (key & (c.P - 1)) * DH;
      uint8_t* dst = ring + slot * Cfg::SLOT;
#pragma unroll
      for (int i = 0; i < (DH + 31) / 32; ++i) {
        const int p = i * 32 + lane;
        if (DH >= 32 || p < DH) {
          copy16_async(dst + k_place<DH>(p) * 16, c.k + at + p * 16);
          copy16_async(dst + 16 * DH + v_place<DH>(p) * 16, c.v + at + p * 16);
        }
      }
    }
    copy_commit();  // a group past the end commits nothing, and counts all the same
  };
  int key = k0 + 16 * warp;
#pragma unroll
  for (int i = 0; i < Cfg::DEPTH - 1; ++i) fetch(key + 64 * i, i);
  int slot = 0;
  for (; key < k1; key += 64) {
    copy_wait<Cfg::DEPTH - 2>();
    __syncwarp();
    KBytes<DH> kb;
    VBytes<DH> vb;
    kb.read(ring + slot * Cfg::SLOT);
    vb.read(ring + slot * Cfg::SLOT);
    {
      // the slot read one group ago is free: every lane has read it
      const int into = slot == 0 ? Cfg::DEPTH - 1 : slot - 1;
      fetch(key + 64 * (Cfg::DEPTH - 1), into);
      slot = slot + 1 == Cfg::DEPTH ? 0 : slot + 1;
    }
    const int pj = (key >> c.p_shift) - j0;
    const float ks = s_page[pj] < 0 ? 0.f : s_ks[pj];
    const float ratio = s_vs[pj] * inv_vmax;
    const int bad = s_page[pj] < 0 ? 0 : 0x7fffffff;  // a refused page has no visible key

    float f[2][4];
    score_tile<DH, FMT, QP, RH>(qa, kb, f);
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2 * RH; ++e) {
        const int kk = key + 8 * n + 2 * t + (e & 1);
        const float x = f[n][e] * (qa.qf[e >> 1] * ks);
        f[n][e] = kk < min(limit[e >> 1], bad) ? x : -INFINITY;
      }
    if (!SH && w.score) {
#pragma unroll
      for (int r = 0; r < RH; ++r)
        if (row0 + g + 8 * r < w.rows) {
          float* sp = w.score + spot(row0, g, 8 * r) * w.ld_score + key + 2 * t;
          *reinterpret_cast<float2*>(sp) = make_float2(f[0][2 * r], f[0][2 * r + 1]);
          *reinterpret_cast<float2*>(sp + 8) = make_float2(f[1][2 * r], f[1][2 * r + 1]);
        }
    }
    // A row's reference moves only when its maximum has outgrown it by more
    // than the slack; all lanes of the warp look at once.
    float m2[RH];
#pragma unroll
    for (int r = 0; r < RH; ++r) {
      m2[r] = fmaxf(fmaxf(f[0][2 * r], f[0][2 * r + 1]), fmaxf(f[1][2 * r], f[1][2 * r + 1]));
      top = fmaxf(top, m2[r] - (ref[r] == -INFINITY ? 0.f : ref[r]) >
                               (ref[r] == -INFINITY ? -INFINITY : KV8_BIAS + KV8_SLACK)
                           ? 1.f
                           : -INFINITY);
    }
    if (__any_sync(0xffffffffu, top > 0.f)) {
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        float m = m2[r];
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        if (m - KV8_BIAS > ref[r]) {
          const float old = ref[r];
          ref[r] = m - KV8_BIAS;
          const float alpha = old == -INFINITY ? 0.f : fast_exp2(old - ref[r]);
          if (old != -INFINITY) {
            sum[r] *= alpha;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              o[n][2 * r] *= alpha;
              o[n][2 * r + 1] *= alpha;
            }
          }
        }
      }
    }
    uint32_t hi[4] = {0u, 0u, 0u, 0u}, lo[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        const float neg = ref[r] == -INFINITY ? 0.f : -ref[r];
        float p[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float x = f[n][2 * r + u];
          const float e = fast_exp2(x + neg);
          sum[r] += e;
          p[u] = x == -INFINITY ? 0.f : e * ratio;
        }
        hi[2 * n + r] = pack_half2(p[0], p[1]);
        if constexpr (PP == 2)
          (RH == 1 ? hi[2 * n + 1] : lo[2 * n + r]) = pack_half2_rest(p[0], p[1], hi[2 * n + r]);
      }
    // Slots past the end, and page 0 where it stands in for a refused page, hold
    // whatever was there (an e4m3 NaN among it): as zeros they cannot reach the
    // product.
    const int stop = min(end, bad);
    if (key + 16 > stop) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (key + (i >> 1) * 8 + 2 * t + (i & 1) >= stop) {
#pragma unroll
          for (int u = 0; u < VBytes<DH>::W; ++u) vb.w[i][u] = 0u;
        }
    }
#pragma unroll
    for (int u = 0; u < VBytes<DH>::W; ++u) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (4 * u + 2 * half >= NT) continue;
        const uint32_t sel = half ? 0x7362 : 0x5140;
        uint32_t b00, b01, b10, b11;
        kv8_cvt4<FMT>(__byte_perm(vb.w[0][u], vb.w[1][u], sel), b00, b01);
        kv8_cvt4<FMT>(__byte_perm(vb.w[2][u], vb.w[3][u], sel), b10, b11);
        const int n = 4 * u + 2 * half;
        if constexpr (PP == 1) {
          mma_f16_16816(o[n], hi[0], hi[1], hi[2], hi[3], b00, b10);
          mma_f16_16816(o[n + 1], hi[0], hi[1], hi[2], hi[3], b01, b11);
        } else {
          float d[2][4];
          if constexpr (RH == 2) {
            mma_f16_16816_first(d[0], lo[0], lo[1], lo[2], lo[3], b00, b10);
            mma_f16_16816_first(d[1], lo[0], lo[1], lo[2], lo[3], b01, b11);
            mma_f16_16816(d[0], hi[0], hi[1], hi[2], hi[3], b00, b10);
            mma_f16_16816(d[1], hi[0], hi[1], hi[2], hi[3], b01, b11);
          } else {
            mma_f16_16816_first(d[0], hi[0], hi[1], hi[2], hi[3], b00, b10);
            mma_f16_16816_first(d[1], hi[0], hi[1], hi[2], hi[3], b01, b11);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              float* to = &o[n + i][e & (OW - 1)];
              f2_unpack(f2_add(f2_pack(to[0], to[1]), f2_pack(d[i][e], d[i][e + 1])), to[0], to[1]);
            }
        }
      }
    }
  }

  // Join the four warps, in the rings' place. Column of accumulator (n, e):
  // (2t + (e & 1)) * NT + n.
  copy_wait<0>();
  __syncthreads();
  float* s_o = reinterpret_cast<float*>(s_ring);  // [4][KV8_ROWS][DH]
#pragma unroll
  for (int r = 0; r < RH; ++r) {
    float l = sum[r];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) {
      s_ref[warp][g + 8 * r] = ref[r];
      s_sum[warp][g + 8 * r] = l;
    }
    float* row = s_o + (warp * KV8_ROWS + g + 8 * r) * DH;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      row[(2 * t) * NT + n] = o[n][2 * r];
      row[(2 * t + 1) * NT + n] = o[n][2 * r + 1];
    }
  }
  __syncthreads();
  for (int i = tid; i < KV8_ROWS * DH; i += 128) {
    const int r = i / DH, d = i - r * DH;
    const int row = row0 + r;
    if (row >= rows) break;
    float top = s_ref[0][r];
#pragma unroll
    for (int u = 1; u < 4; ++u) top = fmaxf(top, s_ref[u][r]);
    float l = 0.f, x = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float a = top == -INFINITY ? 1.f : fast_exp2(s_ref[u][r] - top);
      l += a * s_sum[u][r];
      x += a * s_o[(u * KV8_ROWS + r) * DH + d];
    }
    x *= vmax;
    const int64_t at = spot(row);
    if (!SH && alone) {
      const int tok = row / G;
      const int hq = h * G + row - tok * G;
      kv8_store1(out, b * o_sb + hq * o_sh + tok * o_st + d, dtype, l == 0.f ? 0.f : x / l);
      if (d == 0) {
        const float l2 = l == 0.f ? -INFINITY : top + log2f(l);
        if (lse_out)
          lse_out[(static_cast<int64_t>(b) * c.H * G + hq) * T + tok] = l2 * 0.6931471805599453f;
        if (w.lse) w.lse[at] = l2;
      }
    } else {
      w.part[(at * w.chunks + chunk) * DH + d] = x;
      if (d == 0) {
        w.ref[at * w.chunks + chunk] = top;
        w.sum[at * w.chunks + chunk] = l;
      }
    }
  }
  if constexpr (SH) kv8_end_of_pair(kv8_the(groups...).tiles == 0);
}

// ---------------------------------------------------------------- join

// One CTA per query row: the parts of its chunks, in an order that depends on
// their number only. Latency is what it costs, so every loop has its loads in
// flight together.
constexpr int KV8_JOIN_THREADS = 256;
constexpr int KV8_JOIN_TILE = 1024;  // chunks whose factors shared memory holds

__global__ void __launch_bounds__(KV8_JOIN_THREADS)
    kv8_join_kernel(KV8 c, void* __restrict__ out, int64_t o_sb, int64_t o_sh, int64_t o_st,
                    int dtype, int T, int G, float* __restrict__ lse_out, KV8Work w) {
  __shared__ float s_a[KV8_JOIN_TILE];   // a chunk's factor; 0: it wrote no part
  __shared__ float s_x[KV8_JOIN_THREADS];
  __shared__ float s_m[KV8_JOIN_THREADS / 32], s_l[KV8_JOIN_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x;
  const int bh = blockIdx.y;
  const int b = bh / c.H, h = bh - b * c.H;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t at = (static_cast<int64_t>(bh) * w.rows + row) * w.chunks;
  float top = -INFINITY;
  for (int i = tid; i < w.chunks; i += KV8_JOIN_THREADS) top = fmaxf(top, w.ref[at + i]);
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (lane == 0) s_m[warp] = top;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < KV8_JOIN_THREADS / 32; ++u) top = fmaxf(top, s_m[u]);
  const int parts = KV8_JOIN_THREADS / c.D, d = tid & (c.D - 1), part = tid / c.D;
  float l = 0.f, x = 0.f;
  for (int base = 0; base < w.chunks; base += KV8_JOIN_TILE) {
    const int n = min(w.chunks - base, KV8_JOIN_TILE);
    __syncthreads();
    for (int i = tid; i < n; i += KV8_JOIN_THREADS) {
      const float r = w.ref[at + base + i], sum = w.sum[at + base + i];
      const float a = top == -INFINITY ? 1.f : fast_exp2(r - top);
      l += a * sum;
      // an empty chunk wrote no part (its sum is 0; a NaN sum has a part)
      s_a[i] = r == -INFINITY && sum == 0.f ? 0.f : a;
    }
    __syncthreads();
#pragma unroll 8
    for (int i = part; i < n; i += parts) {
      const float a = s_a[i];
      if (a != 0.f) x += a * w.part[(at + base + i) * c.D + d];
    }
  }
#pragma unroll
  for (int u = 16; u; u >>= 1) l += __shfl_xor_sync(0xffffffffu, l, u);
  if (lane == 0) s_l[warp] = l;
  s_x[tid] = x;
  __syncthreads();
  if (part == 0) {
    for (int u = 1; u < parts; ++u) x += s_x[u * c.D + d];
    l = 0.f;
#pragma unroll
    for (int u = 0; u < KV8_JOIN_THREADS / 32; ++u) l += s_l[u];
    const int tok = row / G;
    const int hq = h * G + row - tok * G;
    kv8_store1(out, b * o_sb + hq * o_sh + tok * o_st + d, dtype, l == 0.f ? 0.f : x / l);
    if (d == 0) {
      const float l2 = l == 0.f ? -INFINITY : top + log2f(l);
      if (lse_out)
        lse_out[(static_cast<int64_t>(b) * c.H * G + hq) * T + tok] = l2 * 0.6931471805599453f;
      if (w.lse) w.lse[static_cast<int64_t>(bh) * w.rows + row] = l2;
    }
  }
}

// The parts of calls with groups: D / 4 lanes a row, so that many rows join at
// once (a CTA a row took 68 us for 30720 rows of 64, 17 for 2048 rows of 17 parts).
// Rows of tokens past counts are zeros.
__global__ void __launch_bounds__(KV8_JOIN_THREADS)
    kv8_join_rows_kernel(KV8 c, void* __restrict__ out, int64_t o_sb, int64_t o_sh, int64_t o_st,
                         int dtype, int vec, const int32_t* __restrict__ counts, int T, int G,
                         float* __restrict__ lse_out, KV8Work w, KV8Groups gr) {
  pdl_launch_dependents();
  pdl_wait();
  const int shift = c.d_shift - 2;                  // lanes of a row, as a power of two
  const int l = threadIdx.x & ((1 << shift) - 1);
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * KV8_JOIN_THREADS + threadIdx.x) >> shift;
  const int64_t all = static_cast<int64_t>(c.B) * c.H * w.rows;
  if (at >= all) return;                            // (whole rows leave together)
  const int bh = static_cast<int>(at / w.rows), row = static_cast<int>(at - static_cast<int64_t>(bh) * w.rows);
  const int b = bh / c.H, h = bh - b * c.H;
  const int tok = row / G, hq = h * G + row - tok * G;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f, top = -INFINITY;
  if (tok < kv8_count(c, counts, b, T)) {
    const float* ref = w.ref + at * w.chunks;
    const float* part_sum = w.sum + at * w.chunks;
    const float* part = w.part + at * w.chunks * c.D + 4 * l;
    // (within its room, whatever a kernel that gave up has left)
    const int used = gr.used ? min(max(gr.used[at], 0), gr.chunks) : gr.chunks;
    // then the parts of the own tokens
    const int n = used + w.chunks - gr.chunks, skip = gr.chunks - used;
#pragma unroll 8
    for (int i = 0; i < n; ++i) top = fmaxf(top, ref[i < used ? i : i + skip]);
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      const int i = j < used ? j : j + skip;
      const float r = ref[i], s = part_sum[i];
      const float a = top == -INFINITY ? 1.f : fast_exp2(r - top);
      sum += a * s;
      // an empty part was not written (its sum is 0; a NaN sum has a part)
      if (!(r == -INFINITY && s == 0.f)) {
        const float4 y = *reinterpret_cast<const float4*>(part + static_cast<int64_t>(i) * c.D);
        x[0] += a * y.x;
        x[1] += a * y.y;
        x[2] += a * y.z;
        x[3] += a * y.w;
      }
    }
  }
  const float f = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int u = 0; u < 4; ++u) x[u] = sum == 0.f ? 0.f : x[u] * f;
  const int64_t o = b * o_sb + hq * o_sh + tok * o_st + 4 * l;
  if (!vec) {
#pragma unroll
    for (int u = 0; u < 4; ++u) kv8_store1(out, o + u, dtype, x[u]);
  } else if (dtype == KF_DT_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + o) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    uint2 y;
    if (dtype == KF_DT_BF16) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(x[0], x[1]), q = __floats2bfloat162_rn(x[2], x[3]);
      y = make_uint2(*reinterpret_cast<const uint32_t*>(&p), *reinterpret_cast<const uint32_t*>(&q));
    } else {
      y = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + o) = y;
  }
  if (l == 0 && lse_out)
    lse_out[(static_cast<int64_t>(b) * c.H * G + hq) * T + tok] =
        sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// What the tensor-memory kernel goes by: each group's shared tokens, rows and
// steps (128 keys of a tile of `tile` rows and a kv head), what each sequence
// shares, (live) the rows of new tokens, and where its CTAs begin. One CTA, a warp a
// group at a time; latency is all it costs, so the groups stay in shared memory.
constexpr int KV8_GROUPS_MAX = 1024;
constexpr int KV8_GROUPS_THREADS = 256;

__global__ void __launch_bounds__(KV8_GROUPS_THREADS)
    kv8_groups_kernel(KV8 c, const int32_t* __restrict__ counts, int T, int G, int per, int tile,
                      KV8Groups gr, int4* __restrict__ group, int64_t* __restrict__ work,
                      int4* __restrict__ record, int ctas, int32_t* __restrict__ of_seq,
                      int32_t* __restrict__ live) {
  constexpr int WARPS = KV8_GROUPS_THREADS / 32;
  __shared__ int4 s_g[KV8_GROUPS_MAX];
  __shared__ int64_t s_work[KV8_GROUPS_MAX + 1];
  __shared__ int s_sum[WARPS], s_share, s_whole;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int before = 0;
  for (int base = 0; base < c.B; base += KV8_GROUPS_THREADS) {
    const int b = base + tid;
    if (b < c.B) of_seq[b] = 0;
    if (!live) continue;
    int sum = b < c.B ? kv8_count(c, counts, b, T) : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    __syncthreads();
    if (lane == 31) s_sum[warp] = sum;
    __syncthreads();
    int all = 0;
    for (int u = 0; u < WARPS; ++u) {
      if (u < warp) sum += s_sum[u];
      all += s_sum[u];
    }
    if (b < c.B) live[b + 1] = before + sum;
    before += all;
  }
  if (live && tid == 0) live[0] = 0;
  __syncthreads();
  for (int n = warp; n < gr.N; n += WARPS) {
    int2 seq = kv8_group(gr, c.B, n);
    int shared = 0;
    if (seq.x < seq.y) {
      const int2 common = kv8_group_tokens(c, gr, counts, T, n, seq);
      shared = common.x;
      seq.x = common.y;    // (sequences before it have no row that is joined)
    }
    const int rows = live ? (live[seq.y] - live[seq.x]) * G : (seq.y - seq.x) * per;
    if (lane == 0) group[n] = s_g[n] = make_int4(shared, rows, seq.x, seq.y);
    if (shared)
      for (int b = seq.x + lane; b < seq.y; b += 32) of_seq[b] = shared;
  }
  __syncthreads();
  auto items_of = [&](const int4& g) -> int {
    return g.x ? (g.y + tile - 1) / tile * c.H : 0;
  };
  auto steps_of = [&](const int4& g) -> int { return (g.x + 127) / 128; };
  if (warp == 0) {
    int64_t total = 0;
    int items = 0;
    for (int n = lane; n < gr.N; n += 32) {
      const int64_t i = items_of(s_g[n]);
      total += i * steps_of(s_g[n]);
      items += static_cast<int>(min(i, static_cast<int64_t>(ctas) + 1));
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    items = __reduce_add_sync(0xffffffffu, items);
    // A CTA's steps: an equal share of all of them, which may end one tile and begin
    // the next; or, where that costs less (a stretch's start and end take about five
    // steps), one stretch each: the shortest that needs no more CTAs than there are.
    const int64_t even = max(static_cast<int64_t>(gr.least), (total + ctas - 1) / ctas);
    int64_t share = even;
    bool whole = false;
    if (items <= ctas) {
      int lo = static_cast<int>(even), hi = max(lo, (gr.max_shared + 127) / 128);
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        int need = 0;
        for (int n = lane; n < gr.N; n += 32)
          need += items_of(s_g[n]) * ((steps_of(s_g[n]) + mid - 1) / mid);
        need = __reduce_add_sync(0xffffffffu, need);
        if (need <= ctas)
          hi = mid;
        else
          lo = mid + 1;
      }
      whole = lo <= even + 5;
      if (whole) share = lo;
    }
    // Steps of the groups before; with one stretch a CTA, those of an item made full.
    int64_t sum = 0;
    for (int base = 0; base < gr.N; base += 32) {
      int64_t x = 0;
      if (base + lane < gr.N) {
        const int4 g = s_g[base + lane];
        const int64_t steps = steps_of(g);
        x = items_of(g) * (whole ? (steps + share - 1) / share * share : steps);
      }
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += o;
      }
      if (base + lane < gr.N) s_work[base + lane + 1] = work[base + lane + 1] = sum + x;
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) {
      s_work[0] = work[0] = 0;
      work[gr.N + 1] = whole ? -share : share;
      // (a share is at most a tile's steps, or an even one; both fit)
      s_share = static_cast<int>(min(share, static_cast<int64_t>(INT32_MAX)));
      s_whole = whole;
    }
  }
  __syncthreads();
  const int share = s_share;
  for (int i = tid; i < ctas; i += KV8_GROUPS_THREADS) {
    const int64_t at = static_cast<int64_t>(i) * share;
    int4 g = make_int4(0, 0, 0, 0), r = make_int4(0, 0, 1, 0);
    if (at < s_work[gr.N]) {
      int lo = 0, hi = gr.N;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_work[mid] <= at)
          lo = mid;
        else
          hi = mid;
      }
      g = s_g[lo];
      const int64_t off = at - s_work[lo];
      r.z = steps_of(g);
      if (s_whole) r.z = (r.z + share - 1) / share * share;
      r.x = static_cast<int>(off / r.z);
      r.y = static_cast<int>(off - static_cast<int64_t>(r.x) * r.z);
      r.w = static_cast<int>(i - (at - r.y) / share);
    }
    record[2 * i] = g;
    record[2 * i + 1] = r;
  }
}

// ---------------------------------------------------------------- weights

// Adds each key's weight to the record, from the scores the split kernel left
// (at most KV8_SPLIT_ROWS rows). One thread per four keys (a page is at least
// 16); the rows are added in order. Measured: 64 x 12 heads, 1k tokens on
// average, 9 us (16 with a key per thread); it waits on a chain of four loads.
constexpr int KV8_WEIGHTS_KEYS = 4 * 128;  // keys of a CTA

__global__ void __launch_bounds__(128)
    kv8_weights_kernel(KV8 c, const int32_t* __restrict__ counts, int T, int G, int max_len,
                       int flags, KV8Work w) {
  __shared__ float s_lse[KV8_SPLIT_ROWS];
  pdl_launch_dependents();
  pdl_wait();
  const int bh = blockIdx.y;
  const int b = bh / c.H, h = bh - b * c.H;
  const int len = kv8_len(c, b);
  const int count = kv8_count(c, counts, b, T);
  const int end = min(kv8_end(c, len, count), max_len);
  if (static_cast<int>(blockIdx.x) * KV8_WEIGHTS_KEYS >= end) return;
  if (threadIdx.x < w.rows)
    s_lse[threadIdx.x] = w.lse[static_cast<int64_t>(bh) * w.rows + threadIdx.x];
  __syncthreads();
  const int key = blockIdx.x * KV8_WEIGHTS_KEYS + 4 * threadIdx.x;
  if (key >= end) return;
  const int page = kv8_page(c, b, key >> c.p_shift);
  if (page < 0) return;
  float* at = c.weight + (static_cast<int64_t>(page) * c.H + h) * c.P + (key & (c.P - 1));
  const bool causal = (flags & KF_KV8_CAUSAL) != 0;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int r = 0; r < w.rows; ++r) {
    const int tok = r / G;
    const float l = s_lse[r];
    // keys of this row: below `limit` (a score past it may not have been written)
    const int limit = tok >= count || l == -INFINITY ? 0 : (causal ? min(len + tok + 1, end) : end);
    if (key >= limit) continue;
    const float4 s = *reinterpret_cast<const float4*>(
        w.score + (static_cast<int64_t>(bh) * w.rows + r) * w.ld_score + key);
    x[0] += fast_exp2(s.x - l);
    if (key + 1 < limit) x[1] += fast_exp2(s.y - l);
    if (key + 2 < limit) x[2] += fast_exp2(s.z - l);
    if (key + 3 < limit) x[3] += fast_exp2(s.w - l);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (key + u < end) at[u] += x[u];
}

}  // namespace kf
