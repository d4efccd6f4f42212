// Shared pieces of the 8-bit key/value cache kernels: the device view of a
// layer's cache, conversions of its codes, and typed loads and stores.
//
// Codes are int8 (scale = amax / 127) or e4m3 (scale = amax / 448), one scale
// for each (page, kv head) and for K and V apart. Both code types are exact in
// fp16 (8 and 4 significant bits), so the attention converts codes to fp16
// without rounding and only q and P are rounded.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kf_common.cuh"

namespace kf {

struct KV8 {
  uint8_t* k;
  uint8_t* v;
  float* scale;   // [pages][H][2]
  float* weight;  // [pages][H][P] or null
  const int32_t* table;
  const int32_t* lens;
  int64_t pages;
  int64_t ld_table;
  int blocks;     // usable table columns
  int B, H, D, P, fmt;
  int p_shift;    // log2 P
  int d_shift;    // log2 D
};

constexpr float KV8_TINY = 1.1754943508222875e-38f;  // 2^-126: smaller scales mean a zero block

__host__ __device__ __forceinline__ float kv8_inv_qmax(int fmt) {
  return fmt == KF_KV8_INT8 ? 1.0f / 127.0f : 1.0f / 448.0f;
}

// Cached tokens of sequence b: lens[b], kept inside the table's reach.
// A length outside it, or a page number outside the pool, is recorded in the
// device status word and never used as an index.
__device__ __forceinline__ int kv8_len(const KV8& c, int b) {
  const int n = __ldg(c.lens + b);
  const int64_t reach = static_cast<int64_t>(c.blocks) << c.p_shift;
  if (n < 0 || n > reach) {
    record_device_status(KF_DEV_BAD_KV_PAGE);
    return n < 0 ? 0 : static_cast<int>(reach);
  }
  return n;
}
// Tokens that a call adds to sequence b (counts null: T). None where its length
// is negative: at position 0 they would fall on tokens that it may hold.
__device__ __forceinline__ int kv8_count(const KV8& c, const int32_t* counts, int b, int T) {
  const int n = counts ? __ldg(counts + b) : T;
  return n < 0 || __ldg(c.lens + b) < 0 ? 0 : (n > T ? T : n);
}
// End of the tokens of sequence b with its counted new ones.
__device__ __forceinline__ int kv8_end(const KV8& c, int len, int count) {
  const int64_t reach = static_cast<int64_t>(c.blocks) << c.p_shift;
  if (len + static_cast<int64_t>(count) > reach) {
    record_device_status(KF_DEV_BAD_KV_PAGE);
    return static_cast<int>(reach);
  }
  return len + count;
}
// Page of block j of sequence b, or -1 (recorded) when the table's entry is
// no page of the pool.
__device__ __forceinline__ int kv8_page(const KV8& c, const int32_t* table, int64_t ld, int b,
                                        int j) {
  const int p = __ldg(table + b * ld + j);
  if (p < 0 || p >= c.pages) {
    record_device_status(KF_DEV_BAD_KV_PAGE);
    return -1;
  }
  return p;
}
__device__ __forceinline__ int kv8_page(const KV8& c, int b, int j) {
  return kv8_page(c, c.table, c.ld_table, b, j);
}

// The same without a branch before the caller's next load, for several lookups
// in flight: page 0 stands in for no page, and *ok tells.
__device__ __forceinline__ int kv8_page_or0(const KV8& c, int b, int j, bool* ok) {
  const int p = __ldg(c.table + b * c.ld_table + j);
  *ok = p >= 0 && p < c.pages;
  return *ok ? p : 0;
}

// ---------------------------------------------------------------- types

__device__ __forceinline__ float kv8_load1(const void* p, int64_t i, int dtype) {
  if (dtype == KF_DT_F32) return static_cast<const float*>(p)[i];
  if (dtype == KF_DT_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void kv8_store1(void* p, int64_t i, int dtype, float x) {
  if (dtype == KF_DT_F32)
    static_cast<float*>(p)[i] = x;
  else if (dtype == KF_DT_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(x);
}
// Four consecutive values; `vec`: the address is aligned for one wide load.
__device__ __forceinline__ void kv8_load4(const void* p, int64_t i, int dtype, bool vec,
                                          float (&x)[4]) {
  if (!vec) {
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = kv8_load1(p, i + u, dtype);
  } else if (dtype == KF_DT_F32) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    float2 a, b;
    if (dtype == KF_DT_BF16) {
      a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x));
      b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
    } else {
      a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
      b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
    }
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
  }
}

// N consecutive values of type DT: 16 bytes.
template <int DT>
struct KV8Type {
  static constexpr int N = DT == KF_DT_F32 ? 4 : 8;
  // The run at element i; `vec`: the address is aligned.
  __device__ __forceinline__ static uint4 load(const void* p, int64_t i, bool vec) {
    if (vec)
      return __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) +
                                                  i * (DT == KF_DT_F32 ? 4 : 2)));
    uint32_t w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if constexpr (DT == KF_DT_F32) {
        w[u] = static_cast<const uint32_t*>(p)[i + u];
      } else {
        const uint16_t* q = static_cast<const uint16_t*>(p) + i + 2 * u;
        w[u] = q[0] | (static_cast<uint32_t>(q[1]) << 16);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ static void values(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if constexpr (DT == KF_DT_F32) {
        x[u] = __uint_as_float(w[u]);
      } else if constexpr (DT == KF_DT_BF16) {
        x[2 * u] = __uint_as_float(w[u] << 16);
        x[2 * u + 1] = __uint_as_float(w[u] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[u]));
        x[2 * u] = f.x;
        x[2 * u + 1] = f.y;
      }
    }
  }
  // The largest magnitude of runs as a bit pattern (an infinity or a NaN is
  // larger than any number): collect() gathers it in a word (two halves for
  // the 16-bit types), bits() turns that into fp32 bits.
  __device__ __forceinline__ static void collect(const uint4& v, uint32_t& m) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int u = 0; u < 4; ++u)
      m = DT == KF_DT_F32 ? max(m, w[u] & 0x7fffffffu) : __vmaxu2(m, w[u] & 0x7fff7fffu);
  }
  __device__ __forceinline__ static uint32_t bits(uint32_t m) {
    if constexpr (DT == KF_DT_F32) return m;
    const uint32_t top = max(m & 0xffffu, m >> 16);
    if constexpr (DT == KF_DT_BF16) return top << 16;
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(top)))) &
           0x7fffffffu;
  }
  // N values to a 16-byte aligned address.
  __device__ __forceinline__ static void store(void* p, int64_t i, const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if constexpr (DT == KF_DT_F32) {
        w[u] = __float_as_uint(x[u]);
      } else if constexpr (DT == KF_DT_BF16) {
        const __nv_bfloat162 y = __floats2bfloat162_rn(x[2 * u], x[2 * u + 1]);
        w[u] = *reinterpret_cast<const uint32_t*>(&y);
      } else {
        const __half2 y = __floats2half2_rn(x[2 * u], x[2 * u + 1]);
        w[u] = *reinterpret_cast<const uint32_t*>(&y);
      }
    }
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p) + i * (DT == KF_DT_F32 ? 4 : 2)) =
        make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// ---------------------------------------------------------------- codes

// Four codes (one word) to two fp16 pairs: exact for both code types.
template <int FMT>
__device__ __forceinline__ void kv8_cvt4(uint32_t w, uint32_t& h01, uint32_t& h23) {
  if constexpr (FMT == KF_KV8_INT8) {
    // byte b + 128 as the low mantissa bits of 1024: 1152 + b, minus 1152
    const uint32_t x = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140);
    const uint32_t b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
    const __half2 s = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    h01 = *reinterpret_cast<const uint32_t*>(&r);
    h23 = *reinterpret_cast<const uint32_t*>(&s);
  } else {
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "mov.b32 {lo, hi}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(h01), "=r"(h23)
        : "r"(w));
  }
}

// Four values to four codes, one word. |x * inv| is at most the largest code
// (but for rounding): inv is 1 / s with s >= max|x| / Qmax, or 0.
template <int FMT>
__device__ __forceinline__ uint32_t kv8_encode4(const float* x, float inv) {
  if constexpr (FMT == KF_KV8_INT8) {
    // x * inv + 1.5 * 2^23: the sum's last place is 1, so it is rounded to the
    // nearest integer (ties to even), whose low byte is the code
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inv), 12582912.f));
    return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
  } else {
    const uint32_t a = __nv_cvt_float2_to_fp8x2(
        make_float2(__fmul_rn(x[0], inv), __fmul_rn(x[1], inv)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t b = __nv_cvt_float2_to_fp8x2(
        make_float2(__fmul_rn(x[2], inv), __fmul_rn(x[3], inv)), __NV_SATFINITE, __NV_E4M3);
    return a | (b << 16);
  }
}
// Four codes (one word) to fp32.
template <int FMT>
__device__ __forceinline__ void kv8_decode4(uint32_t w, float* x) {
  uint32_t a, b;
  kv8_cvt4<FMT>(w, a, b);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a));
  const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&b));
  x[0] = f.x; x[1] = f.y; x[2] = g.x; x[3] = g.y;
}
// Scale of a block whose largest magnitude has the fp32 bits `amax`.
__device__ __forceinline__ float kv8_scale(uint32_t amax, int fmt) {
  const float a = __uint_as_float(amax);
  if (amax >= 0x7f800000u) return __uint_as_float(0x7fc00000u);  // an infinity or a NaN came in
  const float s = __fmul_rn(a, kv8_inv_qmax(fmt));
  return s < KV8_TINY ? 0.f : s;
}
__device__ __forceinline__ float kv8_inverse(float s) { return s > 0.f ? __frcp_rn(s) : 0.f; }

__host__ __device__ __forceinline__ bool kv8_aligned(const void* p, int64_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

}  // namespace kf
