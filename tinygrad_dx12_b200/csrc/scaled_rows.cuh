// scaled_rows.cuh -- block-scaled 8-bit rows: E4M3 codes with a power of two for every 32 values.
//
// A block's scale is the smallest power of two that is not below r = max|x| * (1 / 448), held within
// [2^-100, 2^100]: the largest code lies in (224, 448], nothing is clipped, and 1 / scale is exact, so a
// code is one rounding of x. The arithmetic is the packed cache's for E4M3 with E8M0 scales.
#pragma once

#include "common.cuh"

namespace b200 {
namespace rows8 {

// The scale byte of a block whose largest |x| has the bits `top` (as integers they order like the
// values, with NaN above infinity).
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top > 0x7F800000u) return 255u;
  const uint32_t r = __float_as_uint(__fmul_rn(__uint_as_float(top), 1.0f / 448.0f));
  const uint32_t e = (r + 0x7FFFFFu) >> 23;
  return e < 27u ? 27u : e > 227u ? 227u : e;
}

// 1 / scale; zero for a NaN block (whose codes are zero).
__device__ __forceinline__ float inverse(uint32_t byte) {
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}

// Codes of two values, the first in the low byte; in a NaN block zeros (NaN * 0 would be a NaN code).
__device__ __forceinline__ uint32_t codes2(float a, float b, float inv, bool nan) {
  if (nan) return 0u;
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(a, inv), __fmul_rn(b, inv)), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float code_value(uint8_t c) {
  __nv_fp8_e4m3 v;
  v.__x = c;
  return (float)v;
}

}  // namespace rows8
}  // namespace b200
