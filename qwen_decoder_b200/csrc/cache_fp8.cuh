// A paged cache in 8 bits.  A page of ``ps`` tokens is a row of bytes: the keys [G, ps, d], the values [G, ps, d], e4m3 numbers, then the
// scales [G, ps, 2], of a token's key and value side by side, bytes of exponents as in fp8.cuh with the head's d <= 128 features for a block:
//   k[j] = n_k[j] * 2^(s_k - 127),   v[j] = n_v[j] * 2^(s_v - 127)
// A key or value with an infinity or a NaN has the scale 255 ("no number"), and whoever sees it gets none.
#pragma once
#include "fp8.cuh"

__host__ __device__ __forceinline__ long long c8_page_bytes(int G, int ps, int d) { return (long long)G * ps * (2 * d + 2); }

// what a kernel needs to find a token's rows
struct C8Pages {
  unsigned char* at;
  long long page_bytes;
  int G, ps, d;
};
// row of numbers: which = 0 key, 1 value
__device__ __forceinline__ unsigned char* c8_row(const C8Pages& p, long long page, int which, int g, int offset) {
  return p.at + page * p.page_bytes + ((long long)(which * p.G + g) * p.ps + offset) * p.d;
}
__device__ __forceinline__ unsigned char* c8_scale(const C8Pages& p, long long page, int g, int offset) {
  return p.at + page * p.page_bytes + (long long)2 * p.G * p.ps * p.d + ((long long)g * p.ps + offset) * 2;
}
// 2^(byte - 127) as float32: byte 0 is 2^-127, no normal number; 255 no number
__device__ __forceinline__ float c8_power(unsigned byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23);
}
