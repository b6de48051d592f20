// A paged cache in 8 bits.  A page of ``ps`` tokens is a row of bytes: the keys [G, ps, d], the values [G, ps, d], e4m3 numbers, then the
// scales [G, ps, 2], of a token's key and value side by side, bytes of exponents as in fp8.cuh with the head's d <= 128 features for a block:
//   k[j] = n_k[j] * 2^(s_k - 127),   v[j] = n_v[j] * 2^(s_v - 127)
// A key or value with an infinity or a NaN has the scale 255 ("no number"), and whoever sees it gets none.
#pragma once
#include "fp8.cuh"
#include "tc5_ops.cuh"

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
// Pages as rows of d bytes, [n_pages][2 G ps] of them (the scales behind a page's rows are no part of it), by boxes of 16 rows, swizzled by as
// many bytes as a row has
static bool c8_make_map(CUtensorMap* map, const void* pages, long long n_pages, int G, int ps, int d) {
  TcEncodeFn fn = tc_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)2 * G * ps, (cuuint64_t)n_pages};
  cuuint64_t strides[2] = {(cuuint64_t)d, (cuuint64_t)c8_page_bytes(G, ps, d)};
  cuuint32_t box[3] = {(cuuint32_t)d, 16, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(pages), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
