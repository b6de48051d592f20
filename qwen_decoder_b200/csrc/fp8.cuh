// Rows in 8 bits: e4m3 numbers with a scale to each 128 features of a row, a power of two (the exponent's byte, 127 more than it).
//
// The scale is the smallest with which the block's largest magnitude stays within 448 = 1.75 * 2^8, the largest e4m3 number: for
// m = f * 2^E, 1 <= f < 2, that is 2^(E - 8), or 2^(E - 7) where f > 1.75.  Being a power of two it costs the numbers nothing but the
// choice of 8 bits (a quotient by it is exact), and the tensor cores apply it themselves.  A block of zeros has the scale 1; scales below
// 2^-126 are not used, so that the factor 1 / scale is a normal number; a block that holds an infinity or no number has the scale
// "no number" (255), which makes every sum that takes it none.
#pragma once
#include "common.cuh"

#define FP8_BLOCK 128

// ``m``: the bits of the largest magnitude of a block (magnitudes order as their bits do, infinities and NaN above all numbers)
__device__ __forceinline__ unsigned fp8_scale_byte(unsigned m) {
  if (m >= 0x7f800000u) return 255u;
  if (m == 0) return 127u;
  const int e = (int)(m >> 23) - 8 + ((m & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (unsigned)(e < 1 ? 1 : e);
}
// 1 / scale; what the scale "no number" gives makes every e4m3 number of the block none
__device__ __forceinline__ float fp8_inverse(unsigned byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : (254u - byte) << 23);
}
__device__ __forceinline__ unsigned fp8_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// four numbers to e4m3, to nearest even, the first in the lowest byte
__device__ __forceinline__ unsigned fp8_pack4(float a, float b, float c, float d) {
  unsigned short lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (unsigned)lo | (unsigned)hi << 16;
}
// an e4m3 number
__device__ __forceinline__ float fp8_value(unsigned byte) {
  unsigned h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)byte));
  return __half2float(__ushort_as_half((unsigned short)h));
}
// act(g) u, the quotient and the exponential within 2^-20.  A gate of minus infinity goes as the largest finite one does, to zero.
__device__ __forceinline__ float fp8_gated(float g, float u, int act) {
  float r;
  asm("max.NaN.f32 %0, %0, 0fFF7FFFFF;" : "+f"(g));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + __expf(-qd_gate_arg(g, act))));
  return g * r * u;
}
// the larger magnitude, or no number where one is none
__device__ __forceinline__ float fp8_peak(float a, float b) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(fabsf(b)));
  return a;
}
