// e4m3 codes with a power-of-two exponent per row, the form of the quantised
// KV cache: value = code * 2^(exponent - 127), exponent a byte, 255 marking a
// row that is NaN.  The factor is a power of two, so it adds no rounding of
// its own: the code alone carries the error (at most 2^-4 of the value), and
// one byte per (token, K or V, head) holds it.
#pragma once

#include "common.cuh"

namespace pace {

constexpr int kNanExponent = 255;

// 2^(exponent - 127) in fp32; NaN for kNanExponent.
__device__ __forceinline__ float exponent_factor(uint32_t exponent) {
  if (exponent == 0) return __uint_as_float(0x00400000u);  // 2^-127, subnormal
  if (exponent == (uint32_t)kNanExponent) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(exponent << 23);
}

// Two codes as two fp16 values, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)codes));
  return r;
}

// Four codes (little endian) as floats, exactly.
__device__ __forceinline__ void e4m3x4_to_floats(uint32_t codes, float* f) {
  const uint32_t lo = e4m3x2_to_half2(codes & 0xffffu), hi = e4m3x2_to_half2(codes >> 16);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  f[0] = a.x;
  f[1] = a.y;
  f[2] = b.x;
  f[3] = b.y;
}

// Four floats as codes, round to nearest even, saturating at 448.
__device__ __forceinline__ uint32_t floats_to_e4m3x4(const float* f) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(f[1]), "f"(f[0]));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(f[3]), "f"(f[2]));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// The exponent byte of a row whose largest finite magnitude is `amax`: the
// smallest e >= -126 with amax <= 448 * 2^e, plus 127.  448 = 1.75 * 2^8, so
// with amax = 1.f * 2^(E - 127) it is e = E - 135, one more if 1.f > 1.75.
// A row of zeros so has e = -126, and no weight beside rows that are not.
__device__ __forceinline__ uint32_t row_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(e < 1 ? 1 : e);
}

}  // namespace pace
