// 8-bit floating point (e4m3: 4 bits of exponent, 3 of mantissa, largest value 448) with a scale for each block of 128.
//
// A block x of 128 values (of a row, or of 128 x 128 of a matrix) is held as
//   m = max(max |x|, 2^-100)   (NaN where an x is),   scale = m / 448,   q = e4m3(x * (448 / m)),
// every step one operation in 32 bits, rounded to nearest.  The floor keeps 448 / m finite; a block of zeros is zeros.  A block with an
// infinity has an infinite scale and NaN in that place, one with a NaN is NaN throughout: both make the outputs that they enter NaN.
#pragma once
#include "common.cuh"

constexpr int F8_BLOCK = 128;
constexpr int MOST_EXPERTS = 1024;                                     // of a routed layer: the sort has a thread for each, the products a list

__device__ __forceinline__ float max_nan(float a, float b) {           // NaN where either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
struct BlockScale { float scale, inverse; };
__device__ __forceinline__ BlockScale block_scale(float most) {
  const float m = max_nan(most, 0x1p-100f);
  return {__fdiv_rn(m, 448.f), __fdiv_rn(448.f, m)};
}
// four values as e4m3, the first in the lowest byte
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;\n" : "=h"(lo) : "f"(a), "f"(b));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;\n" : "=h"(hi) : "f"(c), "f"(d));
  return (uint32_t)hi << 16 | lo;
}
