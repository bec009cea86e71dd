// pa_convert.hpp -- eight elements at a time between the activation and cache
// types and fp32, shared by the kernels that write the paged cache.
#pragma once

#include "pa_device.hpp"

namespace pa {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

// Eight source elements (16-byte aligned) as fp32, or as raw 16-bit words
// when source and cache share a 16-bit type.
template <int SRC>
__device__ inline void load8(const void* base, int64_t idx, float (&x)[8]) {
  if constexpr (SRC == kF32) {
    const float4_t a = *reinterpret_cast<const float4_t*>(static_cast<const float*>(base) + idx);
    const float4_t b = *reinterpret_cast<const float4_t*>(static_cast<const float*>(base) + idx + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  } else {
    const u32x4_t r = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(base) + idx);
    if constexpr (SRC == kF16) {
      KvF16::widen(r, x);
    } else {
      KvBF16::widen(r, x);
    }
  }
}

// fp32 -> FP8 E4M3 (OCP, "fn": no infinities) code, round to nearest even,
// saturating at +-448 (the largest finite value; infinities too), NaN ->
// 0x7f, -0 -> 0x80.  Normal range: the fp32 bits rounded to 3 mantissa bits
// and rebiased (exponent bias 127 -> 7); below 2^-6 the code is the integer
// nearest |x| * 2^9 (subnormal steps of 2^-9; 8 is the smallest normal).
__device__ inline uint32_t fp8_e4m3_code(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  const uint32_t sign = (b >> 24) & 0x80u;
  const uint32_t a = b & 0x7fffffffu;
  if (a > 0x7f800000u) return 0x7fu;        // NaN
  if (a >= 0x43e00000u) return sign | 0x7eu;  // |x| >= 448
  if (a >= 0x3c800000u) {                   // |x| >= 2^-6
    const uint32_t r = a + 0x7ffffu + ((a >> 20) & 1u);
    return sign | ((r >> 20) - ((127u - 7u) << 3));
  }
  return sign | (uint32_t)__builtin_rintf(__builtin_bit_cast(float, a) * 512.0f);
}

// x / s rounded to nearest, from r = RN(1 / s): q = RN(x r) is within one ulp
// of x / s, the residual x - q s is exact in one FMA, and RN(q + (x - q s) r)
// is the correctly rounded quotient (Markstein's theorem) while x, r and q
// stay in the normal range.  fast: |r| in [2^-60, 2^60] (host-checked); then
// |x| in [2^-60, 2^61) keeps q normal.  Otherwise (zero, subnormal, huge,
// NaN, infinite operands) the full-precision division is taken.
__device__ inline float div_rn(float x, float s, float r, bool fast) {
  const float q = x * r;
  const uint32_t e = (__builtin_bit_cast(uint32_t, x) >> 23) & 0xffu;  // biased exponent of x
  if (fast && e - 67u <= 120u) return __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
  return (x == 0.0f || x != x) ? q : __fdiv_rn(x, s);
}

template <int DST>
__device__ inline void store8(void* base, int64_t idx, const float (&x)[8]) {
  if constexpr (DST == kFP8) {
    u32x2_t w;
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) nan |= x[e] != x[e];
    if (!nan) {
      // v_cvt_pk_fp8_f32 (round to nearest even) on values clamped to +-448,
      // so that every finite or infinite input saturates as fp8_e4m3_code does.
      float c[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = __builtin_fminf(__builtin_fmaxf(x[e], -448.0f), 448.0f);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * j], c[4 * j + 1], 0, false);
        w[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[4 * j + 2], c[4 * j + 3], lo, true);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        w[j] = fp8_e4m3_code(x[4 * j]) | (fp8_e4m3_code(x[4 * j + 1]) << 8) |
               (fp8_e4m3_code(x[4 * j + 2]) << 16) | (fp8_e4m3_code(x[4 * j + 3]) << 24);
    }
    *reinterpret_cast<u32x2_t*>(static_cast<uint8_t*>(base) + idx) = w;
  } else if constexpr (DST == kF32) {
    float* p = static_cast<float*>(base) + idx;
    *reinterpret_cast<float4_t*>(p) = float4_t{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<float4_t*>(p + 4) = float4_t{x[4], x[5], x[6], x[7]};
  } else {
    u32x4_t w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2_t f = float2_t{x[2 * j], x[2 * j + 1]};
      if constexpr (DST == kF16) {
        w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, half2_t));
      } else {
        w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2_t));
      }
    }
    *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(base) + idx) = w;
  }
}

}  // namespace pa
