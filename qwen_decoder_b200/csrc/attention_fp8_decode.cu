// Attention of single tokens over a paged cache in 8 bits (cache_fp8.cuh):
//
//   z_k = scale 2^(s_k) (q . n_k),   p_k = 2^((z_k - max z) / log 2),   out = sum_k p_k 2^(s_v) n_v / sum_k p_k,   lo <= k <= pos
//
// Bound by the cache's bytes; what a design has to do is keep them coming and turn them into operands cheaply.
//
// * A warp takes 16 keys at a time, straight from memory into registers: keys as the rows of m16n8k16 products, the query heads of the KV
//   head as their 8 columns (two such for groups of 9 to 16).  Both contractions leave the order of their index free, so each thread loads 16
//   contiguous bytes: of the keys, features 16 c.. of rows lane / 4 (and 8 more), with q's fragments in the same order; of the values, 16
//   features of four keys, whose bytes it interleaves by pairs of keys.  Nothing passes through shared memory, and the weights go from the
//   first product's result to the second's operand by one 8x8 transposition of a register.
// * Operands are float16, which an e4m3 number becomes in one instruction and without a rounding.  q is divided by a power of two that
//   brings its largest magnitude below 2^15: of a bfloat16 number down to 2^-25 of that nothing is lost, and what is lost below is 2^-40 of it.
//   A key's scale multiplies its score.
// * A value's scale joins its weight: with w_k = z_k / log 2 + s_v, the weights are 2^(w_k - W), W their own running maximum beside the
//   scores'.  So they are numbers up to 2^8 (both maxima are followed when they grow by more than 2^8), rounded to float16 by 2^-12
//   of themselves, and by 2^-25 of the largest where that is more: 2^-17 of a float16's distance from bfloat16, whatever the scales.  Sums are
//   float32.
// * Work: the keys of all (token, KV head) pairs, in units of 128 (a CTA's eight warps, 16 each), are one list; every CTA takes an equal,
//   contiguous share of it, found from the tokens' positions alone, so that the lengths may differ as they like and a graph's replay needs
//   nothing of the host.  A pair whose keys are one CTA's is finished by it; the others leave their sums in float32, at most two pieces
//   to a CTA, for ``decode_fp8_join``.  No counters are shared between launches.
#include "cache_fp8.cuh"

#include <cuda_fp16.h>

#define DA_WARPS 8
#define DA_THREADS (32 * DA_WARPS)
#define DA_UNIT (16 * DA_WARPS)            // keys
#define DA_TOKENS 1024                     // of a launch
#define DA_GROW 8.0f                       // powers of two by which a maximum grows before it is followed

struct DaArgs {
  const bf16* q; long long ldq;
  bf16* out; long long ldo;
  C8Pages pages;
  int n_pages;
  const int* table; int max_blocks, table_rows;
  const int *token_req, *positions;
  int T, H, gs, window, max_keys;
  float scale_log2e;
  float *part_o, *part_s;                  // [CTA][2][gs][d]; [CTA][2][gs][4]: sum, maximum of scores, of weights
};

__device__ __forceinline__ float da_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned da_halves(unsigned short two) {         // two e4m3 numbers to float16
  unsigned h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
  return h;
}
__device__ __forceinline__ unsigned da_lo(unsigned w) { return da_halves((unsigned short)w); }
__device__ __forceinline__ unsigned da_hi(unsigned w) { return da_halves((unsigned short)(w >> 16)); }
__device__ __forceinline__ unsigned da_pack(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ void da_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned da_transpose(unsigned v) {
  unsigned t;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
  return t;
}
// the cache is written by launches before: no read-only path
__device__ __forceinline__ uint4 da_load16(const unsigned char* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 da_load8(const unsigned char* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ unsigned da_load2(const unsigned char* p) {
  unsigned short v;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p) : "memory");
  return v;
}

// The keys of a token: [lo, hi), and the units that hold them, from the 16 keys on in which lo lies
__device__ __forceinline__ int da_lo_key(const DaArgs& a, int pos) { return a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0; }
__device__ __forceinline__ int da_units(const DaArgs& a, int pos) {
  if (pos < 0) return 1;                                   // no key: a unit all the same, whose CTA writes the zeros
  pos = min(pos, a.max_keys - 1);
  return (pos - (da_lo_key(a, pos) & ~15)) / DA_UNIT + 1;
}
// CTAs that take units, of those there are; CTA i of n takes units [i U / n, (i + 1) U / n)
__device__ __forceinline__ int da_taking(long long U, int ctas) { return (int)(U < ctas ? U : ctas); }
__device__ __forceinline__ int da_first(long long U, int n, int i) { return (int)(U * i / n); }
__device__ __forceinline__ int da_cta_of(long long U, int n, int unit) { return (int)((((long long)unit + 1) * n - 1) / U); }

// units of the tokens before each token (and of all of them) to ``sums``, by the whole block
__device__ __forceinline__ void da_sum_units(const DaArgs& a, int* sums, int* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int t0 = 0; t0 < a.T; t0 += DA_THREADS) {
    const int t = t0 + threadIdx.x;
    const int u = t < a.T ? da_units(a, a.positions[t]) : 0;
    int s = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += v;
    }
    if (lane == 31) scratch[warp] = s;
    __syncthreads();
    int base = before, all = before;
#pragma unroll
    for (int w = 0; w < DA_WARPS; w++) {
      if (w < warp) base += scratch[w];
      all += scratch[w];
    }
    if (t < a.T) sums[t] = base + s - u;
    before = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) sums[a.T] = before;
  __syncthreads();
}

template <int HD, int NT>
__global__ void __launch_bounds__(DA_THREADS, NT == 1 ? 2 : 1) decode_fp8_kernel(const DaArgs a) {
  constexpr int KB = HD / 64;                  // 16-byte pieces of a key's row to a thread
  constexpr int MT = HD / 16;                  // products of 16 features
  constexpr int VW = HD / 32;                  // words of a value's row to a thread
  constexpr int OG = HD / 8 + 4;               // of the sums in shared memory: a thread row's features, and four more against conflicts
  __shared__ int sums[DA_TOKENS + 1], scratch[DA_WARPS];
  __shared__ __align__(16) float o_s[DA_WARPS][8][8 * OG];
  __shared__ float st_s[DA_WARPS][8 * NT][3], f_s[DA_WARPS][8 * NT], fin_s[8 * NT][3];
  pdl_wait();
  pdl_launch_dependents();                     // (after the wait: the join reads positions before its own)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int G = a.pages.G, ps = a.pages.ps;
  da_sum_units(a, sums, scratch);
  const long long U = (long long)sums[a.T] * G;
  const int n = da_taking(U, gridDim.x);
  if ((int)blockIdx.x >= n) return;
  int unit = da_first(U, n, blockIdx.x);
  const int end = da_first(U, n, blockIdx.x + 1);
  for (int piece = 0; unit < end; piece++) {
    // ---- the pair this unit belongs to, and how many of its units are this CTA's
    int t = 0;
    for (int step = DA_TOKENS / 2; step > 0; step >>= 1)
      if (t + step < a.T && (long long)sums[t + step] * G <= unit) t += step;
    const int per = sums[t + 1] - sums[t], of_token = unit - sums[t] * G, kvh = of_token / per, u0 = of_token - kvh * per;
    const int n_units = min(per - u0, end - unit);
    const int pos = min(a.positions[t], a.max_keys - 1), lo = da_lo_key(a, pos), base = lo & ~15;
    const int req = a.token_req[t];
    const int* table = a.table + (long long)min(max(req, 0), a.table_rows - 1) * a.max_blocks;

    // ---- q: columns of both halves of a product's k in the order of the keys' bytes; a thread's column is head g
    unsigned qf[NT][KB][4][2];
    float qs[NT][2];                           // of heads 2 c and 2 c + 1: what a score is multiplied by
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const int h = 8 * n + g;
      float v[KB][16], peak = 0.f;
#pragma unroll
      for (int b = 0; b < KB; b++) {
        uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (h < a.gs) {
          const uint4* src = reinterpret_cast<const uint4*>(a.q + (long long)t * a.ldq + (long long)(kvh * a.gs + h) * HD + 64 * b + 16 * c);
          w[0] = src[0]; w[1] = src[1];
        }
        const unsigned x[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
        for (int i = 0; i < 8; i++) {
          v[b][2 * i] = __uint_as_float(x[i] << 16);
          v[b][2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
          peak = fmaxf(peak, fmaxf(fabsf(v[b][2 * i]), fabsf(v[b][2 * i + 1])));
        }
      }
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
      // the power of two that brings the peak to [2^14, 2^15); its inverse multiplies the scores
      int e = (int)(__float_as_uint(peak) >> 23) - 127 - 14;
      e = peak == 0.f || e == 128 - 14 ? 0 : max(e, -126);      // (an infinity stays one)
      const float down = __uint_as_float((unsigned)(127 - e) << 23), up = __uint_as_float((unsigned)(127 + e) << 23) * a.scale_log2e;
#pragma unroll
      for (int b = 0; b < KB; b++)
#pragma unroll
        for (int s = 0; s < 4; s++) {
          qf[n][b][s][0] = da_pack(v[b][4 * s] * down, v[b][4 * s + 1] * down);
          qf[n][b][s][1] = da_pack(v[b][4 * s + 2] * down, v[b][4 * s + 3] * down);
        }
      qs[n][0] = __shfl_sync(0xffffffffu, up, 8 * c);
      qs[n][1] = __shfl_sync(0xffffffffu, up, 8 * c + 4);
    }

    float o[NT][MT][4], m[NT][2], W[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[n][i][j] = 0.f;
      m[n][0] = m[n][1] = W[n][0] = W[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
    // this warp's 16 keys of unit u: base + 128 u + 16 warp ..; keys that are none read the token's first page
    auto first_key = [&](int u) { return base + u * DA_UNIT + 16 * warp; };
    auto page_of = [&](int key) {
      const int p = key <= pos ? table[key / ps] : 0;
      return min(max(p, 0), a.n_pages - 1);
    };
    uint4 kq[2][KB];
    unsigned vq[4][VW], sc[2];
    auto load_keys = [&](int page, int key) {
      const unsigned char* row = c8_row(a.pages, page, 0, kvh, key % ps);
#pragma unroll
      for (int r = 0; r < 2; r++)
#pragma unroll
        for (int b = 0; b < KB; b++) kq[r][b] = da_load16(row + (g + 8 * r) * HD + 64 * b + 16 * c);
      const unsigned char* scales = c8_scale(a.pages, page, kvh, key % ps);
#pragma unroll
      for (int r = 0; r < 2; r++) sc[r] = da_load2(scales + 2 * (g + 8 * r));
    };
    auto load_values = [&](int page, int key) {
      const unsigned char* row = c8_row(a.pages, page, 1, kvh, key % ps);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const unsigned char* from = row + (2 * c + (j & 1) + 8 * (j >> 1)) * HD + HD / 8 * g;
        if constexpr (HD == 128) {
          const uint4 v = da_load16(from);
          vq[j][0] = v.x; vq[j][1] = v.y; vq[j][2] = v.z; vq[j][3] = v.w;
        } else {
          const uint2 v = da_load8(from);
          vq[j][0] = v.x; vq[j][1] = v.y;
        }
      }
    };
    const int last = u0 + n_units;
    int page = 0;
    if (first_key(u0) <= pos) {
      page = page_of(first_key(u0));
      load_keys(page, first_key(u0));
      load_values(page, first_key(u0));
    }
    for (int u = u0; u < last && first_key(u) <= pos; u++) {
      const int key0 = first_key(u), next = first_key(u + 1);
      const bool more = u + 1 < last && next <= pos;
      const int next_page = more ? page_of(next) : 0;
      // ---- scores
      float z[NT][4];
#pragma unroll
      for (int n = 0; n < NT; n++) z[n][0] = z[n][1] = z[n][2] = z[n][3] = 0.f;
#pragma unroll
      for (int b = 0; b < KB; b++) {
        const unsigned *k0 = &kq[0][b].x, *k1 = &kq[1][b].x;
#pragma unroll
        for (int s = 0; s < 4; s++) {
          const unsigned a0 = da_lo(k0[s]), a1 = da_lo(k1[s]), a2 = da_hi(k0[s]), a3 = da_hi(k1[s]);
#pragma unroll
          for (int n = 0; n < NT; n++) da_mma(z[n], a0, a1, a2, a3, qf[n][b][s][0], qf[n][b][s][1]);
        }
      }
      float fk[2], ev[2];
      bool seen[2];
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const int key = key0 + g + 8 * r;
        seen[r] = key <= pos && key >= lo;
        const unsigned bk = sc[r] & 255u, bv = sc[r] >> 8;
        fk[r] = bv == 255u ? __uint_as_float(0x7fc00000u) : c8_power(bk);       // (a value without a number: its keys' weight is none either)
        ev[r] = (float)((int)bv - 127);
      }
      if (more) load_keys(next_page, next);
      // ---- weights
      float w[NT][4];
      bool grows = false;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          z[n][i] = seen[i >> 1] ? z[n][i] * fk[i >> 1] * qs[n][i & 1] : -INFINITY;
          w[n][i] = z[n][i] + ev[i >> 1];
          grows |= z[n][i] > m[n][i & 1] + DA_GROW || w[n][i] > W[n][i & 1] + DA_GROW;
        }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            float mz = fmaxf(z[n][j], z[n][2 + j]), mw = fmaxf(w[n][j], w[n][2 + j]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              mz = fmaxf(mz, __shfl_xor_sync(0xffffffffu, mz, x));
              mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, x));
            }
            mz = fmaxf(mz, m[n][j]);
            mw = fmaxf(mw, W[n][j]);
            if (mz > m[n][j]) { l[n][j] *= da_exp2(m[n][j] - mz); m[n][j] = mz; }
            if (mw > W[n][j]) {
              const float f = da_exp2(W[n][j] - mw);
              W[n][j] = mw;
#pragma unroll
              for (int i = 0; i < MT; i++) { o[n][i][j] *= f; o[n][i][2 + j] *= f; }
            }
          }
      }
      unsigned pb[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          // (no key seen yet: both maxima are minus infinity, and so is what they are taken from)
          l[n][i & 1] += m[n][i & 1] == -INFINITY && !(z[n][i] != z[n][i]) ? 0.f : da_exp2(z[n][i] - m[n][i & 1]);
          p[i] = W[n][i & 1] == -INFINITY && !(w[n][i] != w[n][i]) ? 0.f : da_exp2(w[n][i] - W[n][i & 1]);
        }
        pb[n][0] = da_transpose(da_pack(p[0], p[1]));
        pb[n][1] = da_transpose(da_pack(p[2], p[3]));
      }
      if (key0 < lo || key0 + 15 > pos) {      // values that nobody may see have the weight zero, and may be no numbers
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int key = key0 + 2 * c + (j & 1) + 8 * (j >> 1);
#pragma unroll
          for (int x = 0; x < VW; x++) vq[j][x] = key < lo || key > pos ? 0u : vq[j][x];
        }
      }
      // ---- values: of a pair of features, the bytes of two keys side by side
#pragma unroll
      for (int x = 0; x < VW; x++)
#pragma unroll
        for (int y = 0; y < 2; y++) {
          const unsigned sel = y ? 0x7362u : 0x5140u;
          const unsigned k01 = __byte_perm(vq[0][x], vq[1][x], sel), k89 = __byte_perm(vq[2][x], vq[3][x], sel);
          const unsigned a0 = da_lo(k01), a1 = da_hi(k01), a2 = da_lo(k89), a3 = da_hi(k89);
#pragma unroll
          for (int n = 0; n < NT; n++) da_mma(o[n][2 * x + y], a0, a1, a2, a3, pb[n][0], pb[n][1]);
        }
      if (more) load_values(next_page, next);
    }

    // ---- the warps' sums together
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], x);
        if (g == 0) {
          float* s = st_s[warp][8 * n + 2 * c + j];
          s[0] = l[n][j]; s[1] = m[n][j]; s[2] = W[n][j];
        }
      }
    __syncthreads();
    if (threadIdx.x < 8 * NT) {
      const int h = threadIdx.x;
      float mz = -INFINITY, mw = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < DA_WARPS; w++) {
        mz = fmaxf(mz, st_s[w][h][1]);
        mw = fmaxf(mw, st_s[w][h][2]);
      }
#pragma unroll
      for (int w = 0; w < DA_WARPS; w++) {
        // (a warp without a key has sums of zero; one whose scores are no numbers has a sum that is none and no maximum)
        sum += st_s[w][h][1] == -INFINITY ? st_s[w][h][0] : st_s[w][h][0] * da_exp2(st_s[w][h][1] - mz);
        f_s[w][h] = st_s[w][h][2] == -INFINITY ? 1.f : da_exp2(st_s[w][h][2] - mw);
      }
      fin_s[h][0] = sum; fin_s[h][1] = mz; fin_s[h][2] = mw;
    }
    const bool whole = n_units == per;
    const long long slot = 2ll * blockIdx.x + (piece ? 1 : 0);      // pieces between a CTA's first and last are whole
#pragma unroll
    for (int n = 0; n < NT; n++) {
      if (n) __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < MT; i += 2)
          *reinterpret_cast<float4*>(&o_s[warp][2 * c + j][g * OG + 2 * i]) = make_float4(o[n][i][j], o[n][i][2 + j], o[n][i + 1][j], o[n][i + 1][2 + j]);
      __syncthreads();
      for (int e = threadIdx.x; e < 8 * HD / 4; e += DA_THREADS) {
        const int h = e / (HD / 4), f = e % (HD / 4) * 4, head = 8 * n + h;
        if (head >= a.gs) continue;
        const int at = f / (HD / 8) * OG + f % (HD / 8);
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < DA_WARPS; w++) {
          const float4 v = *reinterpret_cast<const float4*>(&o_s[w][h][at]);
          const float x = f_s[w][head];
          s.x = fmaf(v.x, x, s.x); s.y = fmaf(v.y, x, s.y); s.z = fmaf(v.z, x, s.z); s.w = fmaf(v.w, x, s.w);
        }
        if (whole) {
          const float sum = fin_s[head][0];
          const float inv = sum == 0.f ? 0.f : da_exp2(fin_s[head][2] - fin_s[head][1]) / sum;
          const __nv_bfloat162 x = __floats2bfloat162_rn(s.x * inv, s.y * inv), y = __floats2bfloat162_rn(s.z * inv, s.w * inv);
          *reinterpret_cast<uint2*>(a.out + (long long)t * a.ldo + (long long)(kvh * a.gs + head) * HD + f) =
              make_uint2(*reinterpret_cast<const unsigned*>(&x), *reinterpret_cast<const unsigned*>(&y));
        } else {
          *reinterpret_cast<float4*>(a.part_o + (slot * a.gs + head) * HD + f) = s;
          if (f == 0) *reinterpret_cast<float4*>(a.part_s + (slot * a.gs + head) * 4) = make_float4(fin_s[head][0], fin_s[head][1], fin_s[head][2], 0.f);
        }
      }
    }
    __syncthreads();                           // shared memory is the next piece's
    unit += n_units;
  }
}

// The pieces of pairs that several CTAs of the launch before (of n_ctas) had: a block to a pair.
template <int HD>
__global__ void __launch_bounds__(DA_THREADS) decode_fp8_join_kernel(const DaArgs a, int n_ctas) {
  __shared__ int sums[DA_TOKENS + 1], scratch[DA_WARPS];
  pdl_launch_dependents();
  da_sum_units(a, sums, scratch);
  const int t = blockIdx.x / a.pages.G, kvh = blockIdx.x % a.pages.G, per = sums[t + 1] - sums[t];
  const long long U = (long long)sums[a.T] * a.pages.G;
  n_ctas = da_taking(U, n_ctas);
  const int from = sums[t] * a.pages.G + kvh * per, c0 = da_cta_of(U, n_ctas, from), c1 = da_cta_of(U, n_ctas, from + per - 1);
  if (c0 == c1) return;
  pdl_wait();
  for (int e = threadIdx.x; e < a.gs * (HD / 4); e += DA_THREADS) {
    const int h = e / (HD / 4), f = e % (HD / 4) * 4;
    float mz = -INFINITY, mw = -INFINITY, sum = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = c0; i <= c1; i++) {
      const long long slot = 2ll * i + (da_first(U, n_ctas, i) < from ? 1 : 0);        // (the CTA's first piece, if it begins here)
      const float4 st = __ldcg(reinterpret_cast<const float4*>(a.part_s + (slot * a.gs + h) * 4));
      const float4 v = __ldcg(reinterpret_cast<const float4*>(a.part_o + (slot * a.gs + h) * HD + f));
      if (st.y > mz) { sum *= da_exp2(mz - st.y); mz = st.y; }
      sum += st.y == -INFINITY ? st.x : st.x * da_exp2(st.y - mz);
      float x = 1.f;
      if (st.z > mw) {
        const float y = da_exp2(mw - st.z);
        s.x *= y; s.y *= y; s.z *= y; s.w *= y;
        mw = st.z;
      } else if (st.z != -INFINITY) {
        x = da_exp2(st.z - mw);
      }
      s.x = fmaf(v.x, x, s.x); s.y = fmaf(v.y, x, s.y); s.z = fmaf(v.z, x, s.z); s.w = fmaf(v.w, x, s.w);
    }
    const float inv = sum == 0.f ? 0.f : da_exp2(mw - mz) / sum;
    const __nv_bfloat162 x = __floats2bfloat162_rn(s.x * inv, s.y * inv), y = __floats2bfloat162_rn(s.z * inv, s.w * inv);
    *reinterpret_cast<uint2*>(a.out + (long long)t * a.ldo + (long long)(kvh * a.gs + h) * HD + f) =
        make_uint2(*reinterpret_cast<const unsigned*>(&x), *reinterpret_cast<const unsigned*>(&y));
  }
}

// CTAs of a launch over T tokens of up to max_keys keys: as many as run at a time, one to a unit at most
static int da_ctas(int T, int G, int gs, int window, int max_keys, int sms) {
  const long long keys = window > 0 && window < max_keys ? window + 15 : max_keys;
  const long long units = (long long)T * G * ((keys + DA_UNIT - 1) / DA_UNIT);
  const long long at_a_time = (long long)(gs > 8 ? 1 : 2) * sms;
  return (int)(units < at_a_time ? units : at_a_time);
}

// float32 numbers of scratch memory that a launch takes
extern "C" long long qd_decode_attention_fp8_scratch(int T, int H, int G, int d, int window, int max_keys, int sms) {
  if (T < 1 || G < 1 || H < 1) return 0;
  const int n = da_ctas(T < DA_TOKENS ? T : DA_TOKENS, G, H / G, window, max_keys, sms);
  return 2ll * n * (H / G) * (d + 4);
}

// q, out: bfloat16 rows [T, H d], ``ldq`` and ``ldo`` apart; table [table_rows, max_blocks] of pages of ps tokens (a multiple of 16), its row of token t is
// token_req[t]; the token sees the keys up to positions[t] (none below zero), the last ``window`` of them if that is positive.  No position may be
// beyond max_keys - 1 (later keys are not seen).
extern "C" int qd_decode_attention_fp8(const void* q, long long ldq, void* out, long long ldo, const void* pages, long long n_pages, const int* table,
                                       int max_blocks, int table_rows, const int* token_req, const int* positions, int T, int H, int G, int d, int ps,
                                       float scale, int window, int max_keys, float* scratch, int sms, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (G < 1 || H < 1 || H % G || H / G > 16 || (d != 64 && d != 128) || ps < 16 || ps % 16 || n_pages < 1 || n_pages > 0x7fffffffll || max_blocks < 1 ||
      table_rows < 1 || max_keys < 1 || window < 0 || (long long)max_blocks * ps < max_keys)
    return QD_ERR_UNSUPPORTED;
  if ((((uintptr_t)q | (uintptr_t)out | (uintptr_t)pages) & 15) || ldq % 8 || ldo % 8) return QD_ERR_UNSUPPORTED;
  const int gs = H / G;
  // the units of a launch fit 31 bits
  if ((long long)(T < DA_TOKENS ? T : DA_TOKENS) * G * (max_keys / DA_UNIT + 2) > 0x7fffffffll) return QD_ERR_UNSUPPORTED;
  for (int t = 0; t < T; t += DA_TOKENS) {
    const int n = T - t < DA_TOKENS ? T - t : DA_TOKENS, ctas = da_ctas(n, G, gs, window, max_keys, sms);
    DaArgs a = {(const bf16*)q + t * ldq, ldq, (bf16*)out + t * ldo, ldo, {(unsigned char*)pages, c8_page_bytes(G, ps, d), G, ps, d}, (int)n_pages,
                table, max_blocks, table_rows, token_req + t, positions + t, n, H, gs, window, max_keys, scale * 1.4426950408889634f,
                scratch, scratch + 2ll * ctas * gs * d};
    if (d == 128) {
      if (gs <= 8) qd_launch(decode_fp8_kernel<128, 1>, dim3(ctas), dim3(DA_THREADS), 0, stream, a);
      else qd_launch(decode_fp8_kernel<128, 2>, dim3(ctas), dim3(DA_THREADS), 0, stream, a);
    } else {
      if (gs <= 8) qd_launch(decode_fp8_kernel<64, 1>, dim3(ctas), dim3(DA_THREADS), 0, stream, a);
      else qd_launch(decode_fp8_kernel<64, 2>, dim3(ctas), dim3(DA_THREADS), 0, stream, a);
    }
    if (max_keys > 1) {
      if (d == 128) qd_launch(decode_fp8_join_kernel<128>, dim3(n * G), dim3(DA_THREADS), 0, stream, a, ctas);
      else qd_launch(decode_fp8_join_kernel<64>, dim3(n * G), dim3(DA_THREADS), 0, stream, a, ctas);
    }
  }
  return qd_last_error();
}
