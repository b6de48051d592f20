// q, k and v of tokens behind their product: bias, the rotation by position, q to bfloat16 rows, k and v to their slots of a cache in 8 bits
// (cache_fp8.cuh).
//
//   x = sum of the parts + bias;   of a pair (a, b) that turns by an angle t: (a cos t - b sin t, a sin t + b cos t)
//   k, v: s = the smallest power of two with max |x| <= 448 s,  n = e4m3(x / s)
//
// q is made in 32 bits and rounded once.  k and v are made in 64 bits up to their numbers: a scale changes where a row's largest magnitude is
// next to 448 times a power of two, and a sum in 32 bits would put it on the other side of that now and then, by the order of its
// additions.  (2,048 tokens of 28 + 4 heads: 8 of 36 rows are such; the kernel takes as long with them in 32 bits.)
//
// A thread has eight neighbouring features (16 bytes of a bfloat16 row) of ``nh`` heads of one token, so that the tables' rows, four times
// a head's bytes, are read once for all of them; rows of few tokens, which wait for their loads alone, have a thread's heads one by one.  The
// pair's other half is a shuffle away.  Bound by its bytes for many tokens, by one trip to memory for few.
#include "cache_fp8.cuh"

#define CW_THREADS 256

struct CwArgs {
  const void* x;
  long long ld, part_step;
  int parts;
  const float* bias;
  bf16* q;
  int T, H, rot, n_pos, nh, q_items, kv_items;       // items: threads' sets of ``nh`` heads of a token
  const float *cos_t, *sin_t;
  const int *positions, *slots;
  int n_slots, write;
  C8Pages pages;
};

template <typename T> __device__ __forceinline__ void cw_load8(const T* p, float (&v)[8]);
template <> __device__ __forceinline__ void cw_load8<float>(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <> __device__ __forceinline__ void cw_load8<bf16>(const bf16* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
// eight features of a head: the parts' sum and the bias
template <typename IN, typename S>
__device__ __forceinline__ void cw_sum(const CwArgs& a, const IN* x, int col, S (&v)[8]) {
  float f[8];
  cw_load8<IN>(x + col, f);
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = (S)f[i];
  for (int p = 1; p < a.parts; p++) {
    cw_load8<IN>(x + p * a.part_step + col, f);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += (S)f[i];
  }
  if (a.bias) {
    cw_load8<float>(a.bias + col, f);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += (S)f[i];
  }
}
// the thread's eight features of a row, turned.  c: its place among the row's threads; mask: theirs
template <bool HALF, typename S>
__device__ __forceinline__ void cw_turn(const CwArgs& a, int c, unsigned mask, const float (&cs)[8], const float (&sn)[8], S (&v)[8]) {
  if (HALF) {
    const int half = a.rot / 16;                       // threads of a half
    const bool turns = c < 2 * half, first = c < half;
    const int other = turns ? (first ? c + half : c - half) : c, lane = (threadIdx.x & 31) - c + other;
    S w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = __shfl_sync(mask, v[i], lane);
    if (turns) {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = first ? v[i] * (S)cs[i] - w[i] * (S)sn[i] : w[i] * (S)sn[i] + v[i] * (S)cs[i];
    }
  } else if (8 * c < a.rot) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const S x = v[2 * i], y = v[2 * i + 1];
      v[2 * i] = x * (S)cs[i] - y * (S)sn[i];
      v[2 * i + 1] = x * (S)sn[i] + y * (S)cs[i];
    }
  }
}
// the byte of the scale of a row whose largest magnitude has the bits m
__device__ __forceinline__ unsigned cw_scale_byte(unsigned long long m) {
  const int e = (int)(m >> 52) - 1023;
  if (e == 1024) return 255u;
  if (m == 0) return 127u;
  const int b = e - 8 + 127 + ((m & 0xfffffffffffffull) > 0xc000000000000ull ? 1 : 0);
  return (unsigned)(b < 1 ? 1 : b > 254 ? 254 : b);
}

template <typename IN, bool HALF>
__global__ void __launch_bounds__(CW_THREADS) rope_kv_write_fp8_kernel(const CwArgs a) {
  pdl_launch_dependents();
  const int per_row = a.pages.d / 8;                   // threads of a row, 8 or 16
  const int c = threadIdx.x % per_row, lane = threadIdx.x & 31;
  const unsigned mask = (per_row == 16 ? 0xffffu : 0xffu) << (lane - c);
  long long item = (long long)blockIdx.x * (CW_THREADS / per_row) + threadIdx.x / per_row;
  // all tokens' q, then k, then v: the threads of a warp do alike
  int kind = 0;
  if (item >= (long long)a.T * a.q_items) {
    item -= (long long)a.T * a.q_items;
    kind = 1 + (item >= (long long)a.T * a.kv_items);
    if (kind == 2) item -= (long long)a.T * a.kv_items;
    if (item >= (long long)a.T * a.kv_items) return;   // (a whole row's threads)
  }
  pdl_wait();
  const int items = kind ? a.kv_items : a.q_items, heads = kind ? a.pages.G : a.H;
  const int t = (int)(item / items), h0 = (int)(item % items) * a.nh;
  const int col0 = (kind == 0 ? 0 : kind == 1 ? a.H : a.H + a.pages.G) * a.pages.d + 8 * c;
  const IN* x = (const IN*)a.x + (long long)t * a.ld;
  float cs[8], sn[8];
  if (kind < 2 && 8 * c < a.rot) {
    const int pos = min(max(a.positions[t], 0), a.n_pos - 1);
    const long long at = (long long)pos * (a.rot / 2) + (HALF ? 8 * (c % (a.rot / 16)) : 4 * c);
    if (HALF) {
      cw_load8<float>(a.cos_t + at, cs);
      cw_load8<float>(a.sin_t + at, sn);
    } else {
      *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(a.cos_t + at);
      *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(a.sin_t + at);
    }
  }
  const int n = min(a.nh, heads - h0);
  if (kind == 0) {
    for (int h = h0; h < h0 + n; h++) {
      float v[8];
      cw_sum<IN, float>(a, x, col0 + h * a.pages.d, v);
      cw_turn<HALF, float>(a, c, mask, cs, sn, v);
      uint4 o;
      unsigned* w = &o.x;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const unsigned*>(&b);
      }
      *reinterpret_cast<uint4*>(a.q + ((long long)t * a.H + h) * a.pages.d + 8 * c) = o;
    }
    return;
  }
  const int slot = a.write ? a.slots[t] : -1;
  if (slot < 0 || slot >= a.n_slots) return;           // (a whole row's threads)
  const int page = slot / a.pages.ps, offset = slot % a.pages.ps;
  for (int h = h0; h < h0 + n; h++) {
    double v[8];
    cw_sum<IN, double>(a, x, col0 + h * a.pages.d, v);
    if (kind == 1) cw_turn<HALF, double>(a, c, mask, cs, sn, v);
    unsigned long long m = 0;                          // (magnitudes order as their bits do)
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, (unsigned long long)__double_as_longlong(v[i]) & 0x7fffffffffffffffull);
    for (int o = per_row / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(mask, m, o));
    const unsigned byte = cw_scale_byte(m);
    const double inv = byte == 255u ? __longlong_as_double(0x7ff8000000000000ll) : __longlong_as_double((long long)(1023 + 127 - (int)byte) << 52);
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = (float)(v[i] * inv);
    *reinterpret_cast<uint2*>(c8_row(a.pages, page, kind - 1, h, offset) + 8 * c) =
        make_uint2(fp8_pack4(f[0], f[1], f[2], f[3]), fp8_pack4(f[4], f[5], f[6], f[7]));
    if (c == 0) c8_scale(a.pages, page, h, offset)[kind - 1] = (unsigned char)byte;
  }
}

// x: rows [T] of (H + 2G) d features ``ld`` apart, bfloat16 or float32, or float32 parts of them ``part_step`` apart; q bfloat16 [T, H d];
// tables [n_pos, rot / 2], none with rot = 0; rot a multiple of 16 (pairs of halves) or of 8 (neighbours); slots of tokens: page * ps + offset, others
// than those of the n_pages are not written.
extern "C" int qd_rope_kv_write_fp8(const void* x, int dtype, long long ld, int parts, long long part_step, const float* bias, void* q, int T,
                                    int H, int G, int d, int rot, int half, const float* cos_t, const float* sin_t, int n_pos,
                                    const int* positions, void* pages, long long n_pages, const int* slots, int ps, int write, int sms,
                                    cudaStream_t stream) {
  if (T <= 0) return 0;
  if ((d != 64 && d != 128) || H < 1 || G < 1 || ps < 1 || parts < 1 || rot < 0 || rot > d || rot % (half ? 16 : 8) || (rot && n_pos < 1) ||
      (dtype != QD_F32 && dtype != QD_BF16) || n_pages * ps > 0x7fffffffll)
    return QD_ERR_UNSUPPORTED;
  if ((((uintptr_t)x | (uintptr_t)bias | (uintptr_t)q | (uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)pages) & 15) || ld % 8 || part_step % 4)
    return QD_ERR_UNSUPPORTED;
  CwArgs a = {x, ld, part_step, parts, bias, (bf16*)q, T, H, rot, n_pos, 1, 0, 0, cos_t, sin_t, positions, slots, (int)(n_pages * ps), write,
              {(unsigned char*)pages, c8_page_bytes(G, ps, d), G, ps, d}};
  const int rows = CW_THREADS / (d / 8);
  // four heads to a thread where that still leaves every multiprocessor two blocks' worth of them
  if ((long long)T * (H + 2 * G) >= 4ll * 2 * sms * rows) a.nh = 4;
  a.q_items = (H + a.nh - 1) / a.nh;
  a.kv_items = (G + a.nh - 1) / a.nh;
  const long long items = (long long)T * (a.q_items + (write ? 2 : 0) * a.kv_items);
  const dim3 grid((unsigned)((items + rows - 1) / rows));
  if (dtype == QD_F32) {
    if (half) qd_launch(rope_kv_write_fp8_kernel<float, true>, grid, dim3(CW_THREADS), 0, stream, a);
    else qd_launch(rope_kv_write_fp8_kernel<float, false>, grid, dim3(CW_THREADS), 0, stream, a);
  } else {
    if (half) qd_launch(rope_kv_write_fp8_kernel<bf16, true>, grid, dim3(CW_THREADS), 0, stream, a);
    else qd_launch(rope_kv_write_fp8_kernel<bf16, false>, grid, dim3(CW_THREADS), 0, stream, a);
  }
  return qd_last_error();
}
