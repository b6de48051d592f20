// Rows in 8 bits: e4m3 numbers with a scale to each 128 features of a row, a power of two (the exponent's byte, 127 more than it).
//
// The scale is the smallest with which the block's largest magnitude stays within 448 = 1.75 * 2^8, the largest e4m3 number: for
// m = f * 2^E, 1 <= f < 2, that is 2^(E - 8), or 2^(E - 7) where f > 1.75.  Being a power of two it costs the numbers nothing but the
// choice of 8 bits (a quotient by it is exact), and the tensor cores apply it themselves.  A block of zeros has the scale 1; scales below
// 2^-126 are not used, so that the factor 1 / scale is a normal number; a block that holds an infinity or no number has the scale
// "no number" (255), which makes every sum that takes it none.
#pragma once
#include "common.cuh"

#define FP8_BLOCK QD_FP8_BLOCK

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
// act(g) u = g / (1 + e^-a) u, a = ``qd_gate_arg(g, act)``, within 6 2^-23 of itself: 2^-22 for the power of two, 2^-23 for the reciprocal, half
// a unit or less for each rounding besides.  An exponent as one float32 would be off by |a| 2^-24 and more (a = -87: 2^-17 of the result, a of
// gelu 2^-15), so what -a / log 2 loses in its rounding goes on as a factor 1 + r (Cody and Waite's reduction), and gelu's a is kept with what
// its own roundings lose.  From a of -87.3 down the result is zero (1 + e^-a has no reciprocal that is a normal number), as of a gate of
// minus infinity.
__device__ __forceinline__ float fp8_gated(float g, float u, int act) {
  const bool gelu = act == QD_ACT_GELU_TANH;
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(g) : "f"(gelu ? -11.f : -88.f));       // (below: zero; products of infinities are none)
  float a = fminf(g, gelu ? 16.f : 128.f), rest = 0.f;                       // (above: e^-a is nothing beside 1)
  if (gelu) {
    // a = g (c + c 0.044715 g^2); c in two parts, the first a multiple of 2^-15, so that the difference from it is exact
    const float t = a * a, s = fmaf(0.071354814f, t, 1.5957642f);
    float lost = fmaf(0.071354814f, t, -(s - 1.5957642f));
    lost = fmaf(0.071354814f, fmaf(a, a, -t), lost);
    lost = fmaf(2.3988325e-9f, t, lost) + 4.9614496e-6f;
    const float whole = a * s;
    rest = fmaf(a, lost, fmaf(a, s, -whole));
    a = fmaxf(whole, -88.f);
  }
  const float p = -1.4426950408889634f * a;                                  // up to 127: a power that is finite
  float r = fmaf(p, 1.9046542e-9f, fmaf(p, -0.69314718f, -a)) - rest, e, inv;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(p));
  e = fmaf(e, r, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(1.0f + e));
  return g * inv * u;
}
// the same in four instructions less, for an epilogue whose code has to be short: within (5 + 1.2 |a|) 2^-23 of itself for silu, (5 + 3.7 |a|) 2^-23
// for gelu where a is negative, 5 2^-23 where it is not: __expf is within 2 + 1.173 |a| units, the reciprocal, the sum and the products within
// 3, and gelu's a, of four roundings and two rounded constants, within 2.5 2^-23 of itself
__device__ __forceinline__ float fp8_gated_short(float g, float u, int act) {
  float inv;
  asm("max.NaN.f32 %0, %0, 0fFF7FFFFF;" : "+f"(g));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(1.0f + __expf(-qd_gate_arg(g, act))));
  return g * inv * u;
}
// the same in float64, of which the rounding to 32 bits is no part
__device__ __forceinline__ double fp8_gated_64(double g, double u, int act) {
  const double a = act == QD_ACT_GELU_TANH ? 1.5957691216057308 * fma(0.044715 * g * g, g, g) : g;
  return fmax(g, -3.4028234663852886e38) / (1.0 + exp(-a)) * u;
}
// the larger magnitude, or no number where one is none
__device__ __forceinline__ float fp8_peak(float a, float b) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(fabsf(b)));
  return a;
}
