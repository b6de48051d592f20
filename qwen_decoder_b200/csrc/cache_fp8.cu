// q, k and v of tokens behind their product: bias, the rotation by position, q to bfloat16 rows, k and v to their slots of a cache in 8 bits
// (cache_fp8.cuh).
//
//   x = sum of the parts + bias;   of a pair (a, b) that turns by an angle t: (a cos t - b sin t, a sin t + b cos t)
//   k, v: s = the smallest power of two with max |x| <= 448 s,  n = e4m3(x / s)
//
// q is made in 32 bits and rounded once.  k and v are made in twice 32 bits up to their numbers: a scale changes where a row's largest magnitude
// is next to 448 times a power of two, and a sum in 32 bits would put it on the other side of that now and then, by the order of its
// additions.  (A pair of float32 numbers, not one of 64 bits, whose instructions take some 20 cycles of a scheduler each: 2,048 tokens of
// 28 + 4 heads 14.7 us with those, 13.4 with pairs, 13.1 without either.)
//
// A thread has eight neighbouring features (16 bytes of a bfloat16 row) of four heads of a token's q, so that the tables' rows, four times
// a head's bytes, are read once for all of them, or of one head of its k or v, whose work is the longest; rows of few tokens, which wait for
// their loads alone, have q's heads one by one, too.  The pair's other half is a shuffle away.  Blocks of the same tokens lie together: a row of
// x is read from one end to the other (2,048 tokens, with x out of the caches, 18.4 us, a set of heads of all tokens at a time 20.4).
//
// One token of 16 + 2 heads, four parts: 2.8 us, which are a launch and three trips to memory behind one another (position, table,
// nothing to overlap them with).  2,048 of 28 + 4: 11.8 us, of which 6 are its 37 MB at the rate of device memory; the rest is the
// wait of each block for its loads, 16 to 20 warps on a multiprocessor.
#include "cache_fp8.cuh"

#define CW_THREADS 128

struct CwArgs {
  const void* x;
  long long ld, part_step;
  int parts;
  const float* bias;
  bf16* q;
  int T, H, rot, n_pos, kv_sets, sets;               // (kv heads to be written; blocks of the same tokens)
  const float *cos_t, *sin_t;
  const int *positions, *slots;
  int n_slots;
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
// A number as the sum of two of 32 bits, to 2^-45 of its terms, after T. J. Dekker, "A floating-point technique for extending the available
// precision", Numerische Mathematik 18 (1971), and D. E. Knuth, The Art of Computer Programming 2, section 4.2.2.
struct CwPair { float hi, lo; };
// the first of them the whole, rounded
__device__ __forceinline__ void cw_round(float& v) {}
__device__ __forceinline__ void cw_round(CwPair& v) {
  const float r = v.hi + v.lo;
  v = {r, v.lo - (r - v.hi)};
}
__device__ __forceinline__ CwPair cw_add(CwPair a, CwPair b) {       // (not yet rounded)
  const float s = a.hi + b.hi, t = s - a.hi;
  return {s, ((a.hi - (s - t)) + (b.hi - t)) + (a.lo + b.lo)};
}
__device__ __forceinline__ CwPair cw_times(CwPair a, float b) {
  const float p = a.hi * b;
  return {p, fmaf(a.lo, b, fmaf(a.hi, b, -p))};
}
__device__ __forceinline__ void cw_set(float x, float& v) { v = x; }
__device__ __forceinline__ void cw_set(float x, CwPair& v) { v = {x, 0.0f}; }
__device__ __forceinline__ void cw_join(float x, float& v) { v += x; }
__device__ __forceinline__ void cw_join(float x, CwPair& v) { v = cw_add(v, {x, 0.0f}); }
__device__ __forceinline__ float cw_two(float x, float a, float y, float b) { return x * a + y * b; }
__device__ __forceinline__ CwPair cw_two(CwPair x, float a, CwPair y, float b) { return cw_add(cw_times(x, a), cw_times(y, b)); }
__device__ __forceinline__ float cw_from(unsigned mask, float v, int lane) { return __shfl_sync(mask, v, lane); }
__device__ __forceinline__ CwPair cw_from(unsigned mask, CwPair v, int lane) { return {__shfl_sync(mask, v.hi, lane), __shfl_sync(mask, v.lo, lane)}; }

// eight features of a head: the first part, which is there, the others and the bias
template <typename IN, typename S>
__device__ __forceinline__ void cw_sum(const CwArgs& a, const IN* x, int col, const float (&first)[8], S (&v)[8]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; i++) cw_set(first[i], v[i]);
#pragma unroll 1
  for (int p = 1; p < a.parts; p++) {
    cw_load8<IN>(x + p * a.part_step + col, f);
#pragma unroll
    for (int i = 0; i < 8; i++) cw_join(f[i], v[i]);
  }
  if (a.bias) {
    cw_load8<float>(a.bias + col, f);
#pragma unroll
    for (int i = 0; i < 8; i++) cw_join(f[i], v[i]);
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
    for (int i = 0; i < 8; i++) w[i] = cw_from(mask, v[i], lane);
    if (turns) {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = cw_two(v[i], cs[i], w[i], first ? -sn[i] : sn[i]);
    }
  } else if (8 * c < a.rot) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const S x = v[2 * i], y = v[2 * i + 1];
      v[2 * i] = cw_two(x, cs[i], y, -sn[i]);
      v[2 * i + 1] = cw_two(y, cs[i], x, sn[i]);
    }
  }
}
// the larger of two magnitudes; one that is no number wins
__device__ __forceinline__ float cw_larger(float m, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
  return r;
}
// the byte of the scale of a row whose largest magnitude is m, or, with ``more``, lies above it by less than half a step
__device__ __forceinline__ unsigned cw_scale_byte(float m, bool more) {
  const unsigned u = __float_as_uint(m), part = u & 0x7fffffu;
  const int e = (int)(u >> 23) - 127;
  if (e == 128) return 255u;
  if (u == 0) return 127u;
  const int b = e - 8 + 127 + (part > 0x600000u || (part == 0x600000u && more) ? 1 : 0);
  return (unsigned)(b < 1 ? 1 : b);
}

template <typename IN, bool HALF, int NH>
__global__ void __launch_bounds__(CW_THREADS) rope_kv_write_fp8_kernel(const CwArgs a) {
  pdl_launch_dependents();
  const int per_row = a.pages.d / 8;                   // threads of a row, 8 or 16
  const int c = threadIdx.x % per_row, lane = threadIdx.x & 31;
  const unsigned mask = (per_row == 16 ? 0xffffu : 0xffu) << (lane - c);
  // a few tokens' blocks lie together: of k, then of v, then of q, whose work is the shortest
  const int group = blockIdx.x / a.sets;
  const int t = group * (CW_THREADS / per_row) + threadIdx.x / per_row;
  int set = blockIdx.x - group * a.sets, kind = 1;
  if (set >= 2 * a.kv_sets) {
    set -= 2 * a.kv_sets;
    kind = 0;
  } else if (set >= a.kv_sets) {
    set -= a.kv_sets;
    kind = 2;
  }
  if (t >= a.T) return;                                // (a whole row's threads)
  pdl_wait();
  const int h0 = kind ? set : set * NH;
  const int col0 = (kind == 0 ? 0 : kind == 1 ? a.H : a.H + a.pages.G) * a.pages.d + 8 * c;
  const IN* x = (const IN*)a.x + (long long)t * a.ld;
  const int slot = kind ? a.slots[t] : -1;
  float f[NH][8], cs[8], sn[8];
  cw_load8<IN>(x + col0 + h0 * a.pages.d, f[0]);       // (all loads before the first use)
  if (kind == 0) {
#pragma unroll
    for (int u = 1; u < NH; u++) cw_load8<IN>(x + col0 + min(h0 + u, a.H - 1) * a.pages.d, f[u]);
  }
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
  if (kind == 0) {
#pragma unroll
    for (int u = 0; u < NH; u++) {
      if (h0 + u >= a.H) break;                        // (a whole row's threads)
      float v[8];
      cw_sum<IN, float>(a, x, col0 + (h0 + u) * a.pages.d, f[u], v);
      cw_turn<HALF, float>(a, c, mask, cs, sn, v);
      uint4 o;
      unsigned* w = &o.x;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const unsigned*>(&b);
      }
      *reinterpret_cast<uint4*>(a.q + ((long long)t * a.H + h0 + u) * a.pages.d + 8 * c) = o;
    }
    return;
  }
  if (slot < 0 || slot >= a.n_slots) return;           // (a whole row's threads)
  const int page = (unsigned)slot / (unsigned)a.pages.ps, offset = slot - page * a.pages.ps;
  CwPair v[8];
  cw_sum<IN, CwPair>(a, x, col0 + h0 * a.pages.d, f[0], v);
  if (kind == 1) cw_turn<HALF, CwPair>(a, c, mask, cs, sn, v);
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    cw_round(v[i]);
    m = cw_larger(m, v[i].hi);
  }
  for (int o = per_row / 2; o > 0; o >>= 1) m = cw_larger(m, __shfl_xor_sync(mask, m, o));
  bool more = false;
  if ((__float_as_uint(m) & 0x7fffffu) == 0x600000u) {               // (the same for a whole row's threads)
#pragma unroll
    for (int i = 0; i < 8; i++) more |= fabsf(v[i].hi) == m && (v[i].hi < 0.0f ? -v[i].lo : v[i].lo) > 0.0f;
    more = __any_sync(mask, more);
  }
  const unsigned byte = cw_scale_byte(m, more);
  // 2^(127 - byte), of a byte up to 247 (that of the largest float32 number); the product is exact
  const float inv = byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float((254u - byte) << 23);
  float n[8];
#pragma unroll
  for (int i = 0; i < 8; i++) n[i] = v[i].hi * inv;
  *reinterpret_cast<uint2*>(c8_row(a.pages, page, kind - 1, h0, offset) + 8 * c) =
      make_uint2(fp8_pack4(n[0], n[1], n[2], n[3]), fp8_pack4(n[4], n[5], n[6], n[7]));
  if (c == 0) c8_scale(a.pages, page, h0, offset)[kind - 1] = (unsigned char)byte;
}

template <typename IN, int NH>
static void cw_launch(int half, dim3 grid, cudaStream_t stream, const CwArgs& a) {
  if (half) qd_launch(rope_kv_write_fp8_kernel<IN, true, NH>, grid, dim3(CW_THREADS), 0, stream, a);
  else qd_launch(rope_kv_write_fp8_kernel<IN, false, NH>, grid, dim3(CW_THREADS), 0, stream, a);
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
  CwArgs a = {x, ld, part_step, parts, bias, (bf16*)q, T, H, rot, n_pos, 0, 0, cos_t, sin_t, positions, slots, (int)(n_pages * ps),
              {(unsigned char*)pages, c8_page_bytes(G, ps, d), G, ps, d}};
  const int rows = CW_THREADS / (d / 8);
  // four heads to a thread where that still leaves every multiprocessor two blocks' worth of them (of 28 + 4 heads, four and one: 64 tokens 3.1 and 2.7 us,
  // 256 3.9 and 3.7, 512 4.6 and 5.8, 2,048 12.1 and 16.4)
  const int nh = (long long)T * (H + 2 * G) >= 4ll * 2 * sms * rows ? 4 : 1;
  a.kv_sets = write ? G : 0;
  a.sets = (H + nh - 1) / nh + 2 * a.kv_sets;
  const long long blocks = ((long long)T + rows - 1) / rows * a.sets;
  if (blocks > 0x7fffffffll) return QD_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)blocks);
  if (nh == 4) {
    if (dtype == QD_F32) cw_launch<float, 4>(half, grid, stream, a);
    else cw_launch<bf16, 4>(half, grid, stream, a);
  } else {
    if (dtype == QD_F32) cw_launch<float, 1>(half, grid, stream, a);
    else cw_launch<bf16, 1>(half, grid, stream, a);
  }
  return qd_last_error();
}
