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
// End of the tokens of sequence b with its counted new ones (counts null: T).
__device__ __forceinline__ int kv8_count(const int32_t* counts, int b, int T) {
  const int n = counts ? __ldg(counts + b) : T;
  return n < 0 ? 0 : (n > T ? T : n);
}
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

// One code to fp32 and back (round to nearest even, saturating).
__device__ __forceinline__ float kv8_decode(uint8_t b, int fmt) {
  if (fmt == KF_KV8_INT8) return static_cast<float>(static_cast<int8_t>(b));
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}
__device__ __forceinline__ uint8_t kv8_encode(float x, int fmt) {
  x = x == x ? x : 0.f;  // only in a block whose scale is NaN already
  if (fmt == KF_KV8_INT8) {
    x = fminf(fmaxf(x, -127.f), 127.f);
    return static_cast<uint8_t>(static_cast<int8_t>(__float2int_rn(x)));
  }
  return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
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
