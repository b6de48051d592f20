// Attention of single tokens over a paged cache in 8 bits (cache_fp8.cuh):
//
//   z_k = scale 2^(s_k) (q . n_k),   p_k = 2^((z_k - max z) / log 2),   out = sum_k p_k 2^(s_v) n_v / sum_k p_k,   lo <= k <= pos
//
// Bound by the cache's bytes; what a design has to do is keep them coming and turn them into operands cheaply.
//
// * A warp takes 16 keys at a time, keys as the rows of m16n8k16 products and the query heads of the KV head as their 8 columns (two such for
//   groups of 9 to 16).  Each warp has a ring of its own of two stages, filled by TMA copies of 16 rows (swizzled, so that what the threads read
//   of the values meets no conflict) and one of their scales; no warp waits for another.  Both contractions leave the order of their
//   index free, so each thread reads 16 contiguous bytes: of the keys, features 16 c.. of rows lane / 4 (and 8 more), with q's fragments in
//   the same order; of the values, 16 features of four keys, whose bytes it interleaves by pairs of keys.  The weights go from the first
//   product's result to the second's operand by one 8x8 transposition of a register.
// * Operands are float16, which an e4m3 number becomes in one instruction and without a rounding.  q is divided by a power of two that
//   brings its largest magnitude below 2^15: of a bfloat16 number down to 2^-25 of that nothing is lost, and what is lost below is 2^-40 of it.
//   A key's scale multiplies its score.
// * A value's scale joins its weight: with w_k = z_k / log 2 + s_v, the weights are 2^(w_k - W), W their own running maximum beside the
//   scores'.  So they are numbers up to 2^8 (both maxima are followed when they grow by more than 2^8), rounded to float16 by 2^-11
//   of themselves, and by 2^-25 of one where that is more (weights below 2^-14), whatever the scales.  Sums are float32.  (w_k is one float32 number: at
//   scores of 2^13 it costs a weight 2^-12 of itself, less than such scores' own errors.)
// * Work, where there is much: the keys of all (token, KV head) pairs, in units of 128 (a CTA's eight warps, 16 each), are one list; every CTA
//   takes a contiguous share of it that takes as long as the others', found from the tokens' positions alone, so that the lengths may differ as they
//   like and a graph's replay needs nothing of the host.  A pair whose keys are one CTA's is finished by it; the others leave their sums in float32, at
//   most two pieces to a CTA, for ``decode_fp8_join``.  No counters are shared between launches.
// * Where there is little, a pair is a cluster's, whose CTAs have equal shares of its units and join over their shared memories.
//
// With 28 + 4 heads of 128: 64 tokens of 8,192 keys 95 us, where their 545 MB take 83 at the rate of device memory (88 in a CTA to each pair, which one
// long token among short ones would have wait for one); 23 of 500 to 4,000 18.4, of which 8.3; one of 100,001 26.3, of which 15.8 (the rest: the launches, the way to the
// first keys, 74 pieces to a pair).  16 + 2 heads, one token of 2,048: 6.8, nothing but latencies (position, page, keys, 16 CTAs' join).
#include "cache_fp8.cuh"
#include "entry_points.h"
#include "tc5_ops.cuh"

#include <cooperative_groups.h>
#include <cuda_fp16.h>

namespace cg = cooperative_groups;

#define DA_WARPS 8
#define DA_THREADS (32 * DA_WARPS)
#define DA_UNIT (16 * DA_WARPS)            // keys
#define DA_STAGES 2                        // of a warp's ring
#define DA_MAX_CLUSTER 16
#define DA_PIECE 3                         // units that a pair costs besides its own (128 tokens of up to 2,000 keys: 48 us without, 39 with 2 or 3, 41 with 4)
#define DA_SNAP 1                          // units next to a pair's ends where it is not cut (64 of up to 300: 14.5 us without)
#define DA_TOKENS 1024                     // of a launch that deals its units out
#define DA_GROW 8.0f                       // powers of two by which a maximum grows before it is followed
#define DA_NONE (-1e30f)                   // the maximum of no scores (a difference to it is a number, as one to minus infinity is not)

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
  int cluster;                             // CTAs to a pair; 0: units dealt out
  int ps_shift;                            // log2 of a page's tokens, or -1
  int* status;
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
// x: byte of a row, y: row of a page, z: page
__device__ __forceinline__ void da_copy_rows(void* dst, const CUtensorMap* map, int y, int z, unsigned long long* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(tc_smem(dst)), "l"(map), "r"(tc_smem(bar)), "r"(0), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void da_copy(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(tc_smem(dst)), "l"(src), "r"(bytes), "r"(tc_smem(bar)) : "memory");
}

// The keys of a token: [lo, hi), and the units that hold them, from the 16 keys on in which lo lies
__device__ __forceinline__ int da_lo_key(const DaArgs& a, int pos) { return a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0; }
__device__ __forceinline__ int da_units(const DaArgs& a, int pos) {
  if (pos < 0) return 1;                                   // no key: a unit all the same, whose CTA writes the zeros
  pos = min(pos, a.max_keys - 1);
  return (pos - (da_lo_key(a, pos) & ~15)) / DA_UNIT + 1;
}
// What is dealt out are the keys' units and DA_PIECE more in front of them for each pair, which stand for what a pair costs besides.  CTAs that take
// units, of those there are: CTA i of n takes those from i U / n on, or from where the pair begins or ends that lies near: a part of a pair costs its sums' way
// through memory.  n is U at most: no two cuts are the same, so every CTA that the join asks for a part of a pair has had one
__device__ __forceinline__ int da_taking(long long U, int ctas, int pairs, int most) {
  // Pairs of as many units each, ``most``: a whole number of CTAs to a pair, so that no cut leaves a little of one (64 tokens of 8,192 keys, 28 + 4 heads,
  // 256 CTAs and 296: 95.5 and 99 us, of 4,000 51.4 and 56.2; of lengths that differ there is no such number, and fewer CTAs take longer: up to 8,000 keys 59.8 and 55.6)
  const int alike = ctas / pairs * pairs;
  if ((long long)most * pairs == U && 5 * alike >= 4 * ctas && alike <= U) return alike;
  return (int)(U < ctas ? U : ctas);
}
__device__ __forceinline__ int da_cut(long long U, int n, int i) { return (int)(U * i / n); }
// (``per``: units of the pair with those in front, ``of_pair``: of them before the cut)
__device__ __forceinline__ int da_snap(int cut, int of_pair, int per) {
  const bool start = per <= DA_PIECE + 2 * DA_SNAP + 1 ? 2 * of_pair <= per : of_pair <= DA_PIECE + DA_SNAP;
  if (start) return cut - of_pair;
  return per <= DA_PIECE + 2 * DA_SNAP + 1 || per - of_pair <= DA_SNAP ? cut + per - of_pair : cut;
}
// The CTAs that units [from, from + per) of a pair are cut between: the first of them and the last (none: not less)
__device__ __forceinline__ int2 da_cut_by(long long U, int n, int from, int per) {
  const long long a = (long long)from + DA_PIECE + DA_SNAP + 1, b = (long long)from + per - DA_SNAP;            // cuts in [a, b)
  if (a >= b) return make_int2(0, 0);
  return make_int2((int)((a * n + U - 1) / U) - 1, (int)((b * n + U - 1) / U) - 1);
}

// The list of all tokens' units.  Up to 32 tokens: in the registers of every warp, a lane to a token; more: in shared memory, made by the
// whole block.
struct DaList {
  int few, T, most, before, units, pos;        // most: units that a token has; of this lane's token: units of those before it, its own, its position
  const int *sums, *positions;
  __device__ __forceinline__ int all() const { return few ? __shfl_sync(0xffffffffu, before + units, T - 1) : sums[T]; }
  // the token that unit ``u`` of ``G`` times the list is of: a whole warp looks, at every 32nd of them and then at 32 (one after the other by halves it
  // was 900 cycles, at the beginning of every CTA)
  __device__ __forceinline__ int token(int u, int G) const {
    const int lane = threadIdx.x & 31;
    if (few) return __popc(__ballot_sync(0xffffffffu, lane < T && before * G <= u)) - 1;
    const int from = 32 * (__popc(__ballot_sync(0xffffffffu, 32 * lane < T && sums[min(32 * lane, T)] * G <= u)) - 1);
    return from + __popc(__ballot_sync(0xffffffffu, from + lane < T && sums[min(from + lane, T)] * G <= u)) - 1;
  }
  __device__ __forceinline__ int units_before(int t) const { return few ? __shfl_sync(0xffffffffu, before, t) : sums[t]; }
  __device__ __forceinline__ int units_of(int t) const { return few ? __shfl_sync(0xffffffffu, units, t) : sums[t + 1] - sums[t]; }
  __device__ __forceinline__ int position(int t) const { return few ? __shfl_sync(0xffffffffu, pos, t) : positions[t]; }
};
template <int THREADS>
__device__ __forceinline__ DaList da_list(const DaArgs& a, int* sums, int* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto scan = [&](int s) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += v;
    }
    return s;
  };
  DaList list;
  list.few = a.T <= 32;
  list.T = a.T;
  list.sums = sums;
  list.positions = a.positions;
  if (list.few) {
    list.pos = lane < a.T ? a.positions[lane] : -1;
    list.units = lane < a.T ? da_units(a, list.pos) + DA_PIECE : 0;
    list.before = scan(list.units) - list.units;
    list.most = (int)__reduce_max_sync(0xffffffffu, (unsigned)list.units);
    return list;
  }
  int before = 0;
  unsigned most = 0;
  for (int t0 = 0; t0 < a.T; t0 += THREADS) {
    const int t = t0 + threadIdx.x;
    const int u = t < a.T ? da_units(a, a.positions[t]) + DA_PIECE : 0;
    const int s = scan(u);
    most = max(most, __reduce_max_sync(0xffffffffu, (unsigned)u));
    if (lane == 31) scratch[warp] = s;
    __syncthreads();
    int base = before, all = before;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
      if (w < warp) base += scratch[w];
      all += scratch[w];
    }
    if (t < a.T) sums[t] = base + s - u;
    before = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) sums[a.T] = before;
  if (lane == 0) scratch[warp] = (int)most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; w++) most = max(most, (unsigned)scratch[w]);
  list.most = (int)most;
  return list;
}

// What the sum of weighted values is multiplied by, one after the other (together they may be no normal number): 1 / sum, 2^(mw - mz)
__device__ __forceinline__ float2 da_inverse(float sum, float mz, float mw) {
  float up;
  asm("ex2.approx.f32 %0, %1;" : "=f"(up) : "f"(mw - mz));
  return make_float2(sum == 0.f ? 0.f : 1.f / sum, up);
}

// Sums of pieces of a pair together: of the exponentials (their sum and maximum), of the weighted values (and their maximum).
struct DaJoin {
  float sum, mz, mw;
  float4 s;
  __device__ __forceinline__ void none() { sum = 0.f; mz = mw = DA_NONE; s = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void add(float l, float m, float W, float4 v) {
    const float z = fmaxf(mz, m), w = fmaxf(mw, W), a = da_exp2(mw - w), b = da_exp2(W - w);
    sum = sum * da_exp2(mz - z) + l * da_exp2(m - z);
    s.x = fmaf(v.x, b, s.x * a); s.y = fmaf(v.y, b, s.y * a); s.z = fmaf(v.z, b, s.z * a); s.w = fmaf(v.w, b, s.w * a);
    mz = z;
    mw = w;
  }
  __device__ __forceinline__ float2 inverse() const { return da_inverse(sum, mz, mw); }
};
__device__ __forceinline__ void da_store(bf16* to, float4 s, float2 by) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(s.x * by.x * by.y, s.y * by.x * by.y), y = __floats2bfloat162_rn(s.z * by.x * by.y, s.w * by.x * by.y);
  *reinterpret_cast<uint2*>(to) = make_uint2(*reinterpret_cast<const unsigned*>(&x), *reinterpret_cast<const unsigned*>(&y));
}

// a CTA's part of a pair's keys
struct DaPiece {
  int t, kvh, per, u0, n;                      // token, KV head, units of the pair, the first and how many
  int pos, lo;                                 // keys [lo, pos]; units from the 16 keys on in which lo lies
  const int* table;
};
__device__ __forceinline__ void da_piece_keys(const DaArgs& a, DaPiece& p, int pos, int request) {
  p.pos = max(min(pos, a.max_keys - 1), -1);     // (what is far below zero as well: differences to it fit 32 bits)
  p.lo = da_lo_key(a, p.pos);
  p.table = a.table + (long long)min(max(request, 0), a.table_rows - 1) * a.max_blocks;
}

template <int HD, int NT, bool CLUSTER>
__global__ void __launch_bounds__(DA_THREADS, NT == 1 ? 2 : 1) decode_fp8_kernel(const __grid_constant__ CUtensorMap map, const DaArgs a) {
  constexpr int KB = HD / 64;                  // 16-byte pieces of a key's row to a thread
  constexpr int MT = HD / 16;                  // products of 16 features
  constexpr int VW = HD / 32;                  // words of a value's row to a thread
  constexpr int OG = HD / 8 + 4;               // of the sums in shared memory: a thread row's features, and four more against conflicts
  constexpr int ROWS = 16 * HD, STAGE = 2 * ROWS;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  unsigned char* ring = smem_raw + ((1024 - (tc_smem(smem_raw) & 1023)) & 1023);           // [warp][stage][key, value][16][HD]
  float* o_s = reinterpret_cast<float*>(ring + DA_WARPS * DA_STAGES * STAGE);              // [warp][8][8 OG]
  __shared__ __align__(16) unsigned char scales_s[DA_WARPS][DA_STAGES][32];
  __shared__ unsigned long long full[DA_WARPS][DA_STAGES];
  __shared__ int sums[CLUSTER ? 1 : DA_TOKENS + 1], scratch[DA_WARPS], dead;
  __shared__ float st_s[DA_WARPS][8 * NT][3], f_s[DA_WARPS][8 * NT], fin_s[8 * NT][4];
  __shared__ __align__(16) float res_s[CLUSTER ? 8 * NT * HD : 4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int G = a.pages.G, ps = a.pages.ps;
  if (threadIdx.x == 0) dead = 0;
  if (lane == 0) {
    for (int s = 0; s < DA_STAGES; s++) tc_bar_init(&full[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();                     // (after the wait: the join reads positions before its own)

  // ---- this CTA's first piece
  DaPiece p;
  DaList list;
  int unit = 0, end = 0;
  if constexpr (CLUSTER) {
    const int pair = blockIdx.x / a.cluster, rank = blockIdx.x % a.cluster;
    p.t = pair / G;
    p.kvh = pair % G;
    da_piece_keys(a, p, a.positions[p.t], a.token_req[p.t]);
    p.per = da_units(a, p.pos);
    p.u0 = p.per * rank / a.cluster;
    p.n = p.per * (rank + 1) / a.cluster - p.u0;
  } else {
    list = da_list<DA_THREADS>(a, sums, scratch);
    const long long U = (long long)list.all() * G;
    const int n = da_taking(U, gridDim.x, a.T * G, list.most);
    if ((int)blockIdx.x >= n) return;
    auto first_of = [&](int i) {
      const int cut = da_cut(U, n, i);
      if (i == n) return cut;
      const int t = list.token(cut, G), per = list.units_of(t);
      return da_snap(cut, (cut - list.units_before(t) * G) % per, per);
    };
    unit = first_of(blockIdx.x);
    end = first_of(blockIdx.x + 1);
    if (unit == end) return;
  }
  __syncthreads();                             // (``dead`` and the barriers are there)
  // the piece that begins at ``unit``, but for its keys; ``unit`` moves on behind it
  auto piece_to = [&](DaPiece& q, int of_pair) {
    const int n = min(q.per + DA_PIECE - of_pair, end - unit);
    q.u0 = max(of_pair - DA_PIECE, 0);
    q.n = of_pair + n - DA_PIECE - q.u0;
    unit += n;
  };
  auto piece_at = [&]() {
    DaPiece q;
    q.t = list.token(unit, G);
    q.per = list.units_of(q.t) - DA_PIECE;
    const int of_token = unit - list.units_before(q.t) * G;
    q.kvh = of_token / (q.per + DA_PIECE);
    piece_to(q, of_token - q.kvh * (q.per + DA_PIECE));
    return q;
  };
  auto piece_after = [&](const DaPiece& p) {   // (of the same token: with its keys)
    DaPiece q = p;
    if (++q.kvh == G) {
      q.kvh = 0;
      q.t++;
      q.per = list.units_of(q.t) - DA_PIECE;
    }
    piece_to(q, 0);
    return q;
  };
  if constexpr (!CLUSTER) {
    p = piece_at();
    da_piece_keys(a, p, list.position(p.t), a.token_req[p.t]);
  }
  // this warp's 16 keys of unit u: base + 128 u + 16 warp ..
  auto first_key = [&](const DaPiece& p, int u) { return (p.lo & ~15) + u * DA_UNIT + 16 * warp; };
  auto chunks_of = [&](const DaPiece& p) {
    const int left = p.pos - first_key(p, p.u0);
    return left < 0 ? 0 : min(p.n, left / DA_UNIT + 1);
  };
  int done = 0;                                // chunks that this warp has taken: the ring's turn
  auto page_of = [&](const DaPiece& p, int i) {
    const int key = first_key(p, p.u0 + i);
    return p.table[a.ps_shift >= 0 ? key >> a.ps_shift : key / ps];
  };
  // chunk i of the piece into the stage of turn ``done + ahead``
  auto request = [&](const DaPiece& p, int i, int ahead, int page) {
    if (lane == 0) {
      page = min(max(page, 0), a.n_pages - 1);
      const int s = (done + ahead) % DA_STAGES, key = first_key(p, p.u0 + i), offset = a.ps_shift >= 0 ? key & (ps - 1) : key % ps;
      unsigned char* to = ring + (warp * DA_STAGES + s) * STAGE;
      unsigned long long* bar = &full[warp][s];
      tc_expect_tx(bar, STAGE + 32);
      da_copy_rows(to, &map, p.kvh * ps + offset, page, bar);
      da_copy_rows(to + ROWS, &map, (G + p.kvh) * ps + offset, page, bar);
      da_copy(scales_s[warp][s], c8_scale(a.pages, page, p.kvh, offset), 32, bar);
    }
  };
  int chunks = chunks_of(p);
  for (int i = 0; i < min(chunks, DA_STAGES); i++) request(p, i, i, page_of(p, i));

  for (int piece = 0;; piece++) {
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
          const uint4* src = reinterpret_cast<const uint4*>(a.q + (long long)p.t * a.ldq + (long long)(p.kvh * a.gs + h) * HD + 64 * b + 16 * c);
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
      m[n][0] = m[n][1] = W[n][0] = W[n][1] = DA_NONE;
      l[n][0] = l[n][1] = 0.f;
    }
    int page_next = chunks > DA_STAGES ? page_of(p, DA_STAGES) : 0;
    // What the next piece's first requests need, each a trip to memory that would otherwise begin with this one's end: its token's position
    // and request now, its first pages after this piece's first keys
    bool more = false;
    DaPiece next = p;
    int next_pages[DA_STAGES] = {0, 0};
    if constexpr (!CLUSTER) {
      more = unit < end;
      if (more) {
        next = piece_after(p);
        if (next.t != p.t) {
          next.pos = list.position(next.t);
          next.lo = a.token_req[next.t];       // (until its pages are looked up)
        }
      }
    }
    auto next_pages_of = [&]() {
      if (next.t != p.t) da_piece_keys(a, next, next.pos, next.lo);
      const int n = chunks_of(next);
#pragma unroll
      for (int i = 0; i < DA_STAGES; i++) next_pages[i] = i < n ? page_of(next, i) : 0;
    };
    if (more && chunks == 0) next_pages_of();
    for (int i = 0; i < chunks; i++, done++) {
      const int s = done % DA_STAGES, key0 = first_key(p, p.u0 + i);
      if (!tc_wait(&full[warp][s], done / DA_STAGES & 1, &dead) && lane == 0) atomicCAS(a.status, 0, 1);
      const unsigned char* ks = ring + (warp * DA_STAGES + s) * STAGE;
      const unsigned char* vs = ks + ROWS;
      // ---- scores, of the two halves of the features apart
      float z[KB][NT][4];
#pragma unroll
      for (int b = 0; b < KB; b++) {
        uint4 kq[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const int row = g + 8 * r, place = HD == 128 ? (4 * b + c) ^ g : c ^ (g >> 1 & 3);
          kq[r] = *reinterpret_cast<const uint4*>(ks + row * HD + 16 * place);
        }
        const unsigned *k0 = &kq[0].x, *k1 = &kq[1].x;
#pragma unroll
        for (int n = 0; n < NT; n++) z[b][n][0] = z[b][n][1] = z[b][n][2] = z[b][n][3] = 0.f;
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const unsigned a0 = da_lo(k0[x]), a1 = da_lo(k1[x]), a2 = da_hi(k0[x]), a3 = da_hi(k1[x]);
#pragma unroll
          for (int n = 0; n < NT; n++) da_mma(z[b][n], a0, a1, a2, a3, qf[n][b][x][0], qf[n][b][x][1]);
        }
      }
      const bool border = key0 < p.lo || key0 + 15 > p.pos;     // some of the keys may be seen by nobody
      float fk[2], ev[2];
      {
        const unsigned b0 = *reinterpret_cast<const unsigned short*>(scales_s[warp][s] + 2 * g);
        const unsigned b1 = *reinterpret_cast<const unsigned short*>(scales_s[warp][s] + 2 * g + 16);
        fk[0] = __uint_as_float(b0 << 23 & 0x7f800000u);        // (as c8_power but for the bytes 0 and 255)
        fk[1] = __uint_as_float(b1 << 23 & 0x7f800000u);
        ev[0] = (float)((int)(b0 >> 8) - 127);
        ev[1] = (float)((int)(b1 >> 8) - 127);
        const unsigned two = b0 | b1 << 16;                     // a byte of 0 or 255: (byte + 1) & 254 is 0
        const unsigned odd = __vadd4(two, 0x01010101u) & 0xfefefefeu;
        if (__any_sync(0xffffffffu, __vcmpeq4(odd, 0u))) {
          fk[0] = b0 >> 8 == 255u ? c8_power(255u) : c8_power(b0 & 255u);      // (a value without a number: its key's weight is none either)
          fk[1] = b1 >> 8 == 255u ? c8_power(255u) : c8_power(b1 & 255u);
        }
      }
      // ---- weights: scores, and with the values' exponents; d and w: above the references of their maxima
      float d[NT][4], w[NT][4];
      bool grows = false;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++)            // (the scales first: a large one times a score before the query's small one may leave float32)
          z[0][n][j] = (KB == 2 ? z[0][n][j] + z[KB - 1][n][j] : z[0][n][j]) * (fk[j >> 1] * qs[n][j & 1]);
      if (border) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int key = key0 + g + 8 * (j >> 1);
            if (key > p.pos || key < p.lo) z[0][n][j] = -INFINITY;
          }
      }
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          d[n][j] = z[0][n][j] - m[n][j & 1];
          w[n][j] = z[0][n][j] + ev[j >> 1] - W[n][j & 1];
          grows |= fmaxf(d[n][j], w[n][j]) > DA_GROW;
        }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            float mz = fmaxf(z[0][n][j], z[0][n][2 + j]), mw = fmaxf(z[0][n][j] + ev[0], z[0][n][2 + j] + ev[1]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              mz = fmaxf(mz, __shfl_xor_sync(0xffffffffu, mz, x));
              mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, x));
            }
            if (mz > m[n][j]) { l[n][j] *= da_exp2(m[n][j] - mz); m[n][j] = mz; }
            if (mw > W[n][j]) {
              const float f = da_exp2(W[n][j] - mw);
              W[n][j] = mw;
#pragma unroll
              for (int i = 0; i < MT; i++) { o[n][i][j] *= f; o[n][i][2 + j] *= f; }
            }
#pragma unroll
            for (int x = 0; x < 2; x++) {
              d[n][2 * x + j] = z[0][n][2 * x + j] - m[n][j];
              w[n][2 * x + j] = z[0][n][2 * x + j] + ev[x] - W[n][j];
            }
          }
      }
      unsigned pb[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float q[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          l[n][j & 1] += da_exp2(d[n][j]);
          q[j] = da_exp2(w[n][j]);
        }
        pb[n][0] = da_transpose(da_pack(q[0], q[1]));
        pb[n][1] = da_transpose(da_pack(q[2], q[3]));
      }
      // ---- values: of a pair of features, the bytes of two keys side by side
      unsigned vq[4][VW];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int row = 2 * c + (j & 1) + 8 * (j >> 1);
        if constexpr (HD == 128) {
          const uint4 v = *reinterpret_cast<const uint4*>(vs + row * HD + 16 * (g ^ (row & 7)));
          vq[j][0] = v.x; vq[j][1] = v.y; vq[j][2] = v.z; vq[j][3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(vs + row * HD + 16 * ((g >> 1) ^ (row >> 1 & 3)) + 8 * (g & 1));
          vq[j][0] = v.x; vq[j][1] = v.y;
        }
      }
      __syncwarp();                            // the stage has been read
      if (i + DA_STAGES < chunks) {
        request(p, i + DA_STAGES, DA_STAGES, page_next);
        if (i + DA_STAGES + 1 < chunks) page_next = page_of(p, i + DA_STAGES + 1);
      }
      if (!CLUSTER && i == 0 && more) next_pages_of();
      if (border) {                            // values that nobody may see have the weight zero, and may be no numbers
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int key = key0 + 2 * c + (j & 1) + 8 * (j >> 1);
#pragma unroll
          for (int x = 0; x < VW; x++) vq[j][x] = key < p.lo || key > p.pos ? 0u : vq[j][x];
        }
      }
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
    }

    // ---- the next piece's first keys are on their way while this one's sums come together
    if constexpr (!CLUSTER) {
      if (more) {
        chunks = chunks_of(next);
#pragma unroll
        for (int i = 0; i < DA_STAGES; i++)
          if (i < chunks) request(next, i, i, next_pages[i]);
      }
    }
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
    const bool whole = p.n == p.per;
    const long long slot = 2ll * blockIdx.x + (piece ? 1 : 0);      // pieces between a CTA's first and last are whole
#pragma unroll
    for (int n = 0; n < NT; n++) {
      if (n) __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < MT; i += 2)
          *reinterpret_cast<float4*>(o_s + (warp * 8 + 2 * c + j) * (8 * OG) + g * OG + 2 * i) =
              make_float4(o[n][i][j], o[n][i][2 + j], o[n][i + 1][j], o[n][i + 1][2 + j]);
      __syncthreads();
      if (n == 0) {
        if (threadIdx.x < 8 * NT) {
          const int h = threadIdx.x;
          float mz = DA_NONE, mw = DA_NONE, sum = 0.f;
#pragma unroll
          for (int w = 0; w < DA_WARPS; w++) {
            mz = fmaxf(mz, st_s[w][h][1]);
            mw = fmaxf(mw, st_s[w][h][2]);
          }
#pragma unroll
          for (int w = 0; w < DA_WARPS; w++) {
            // (a warp without a key has sums of zero; one whose scores are no numbers has a sum that is none)
            sum += st_s[w][h][0] * da_exp2(st_s[w][h][1] - mz);
            f_s[w][h] = da_exp2(st_s[w][h][2] - mw);
          }
          fin_s[h][0] = sum; fin_s[h][1] = mz; fin_s[h][2] = mw;
        }
        __syncthreads();
      }
      for (int e = threadIdx.x; e < 8 * HD / 4; e += DA_THREADS) {
        const int h = e / (HD / 4), f = e % (HD / 4) * 4, head = 8 * n + h;
        if (head >= a.gs) continue;
        const int at = f / (HD / 8) * OG + f % (HD / 8);
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < DA_WARPS; w++) {
          const float4 v = *reinterpret_cast<const float4*>(o_s + (w * 8 + h) * (8 * OG) + at);
          const float x = f_s[w][head];
          s.x = fmaf(v.x, x, s.x); s.y = fmaf(v.y, x, s.y); s.z = fmaf(v.z, x, s.z); s.w = fmaf(v.w, x, s.w);
        }
        if (CLUSTER) {
          *reinterpret_cast<float4*>(res_s + head * HD + f) = s;
        } else if (whole) {
          da_store(a.out + (long long)p.t * a.ldo + (long long)(p.kvh * a.gs + head) * HD + f, s, da_inverse(fin_s[head][0], fin_s[head][1], fin_s[head][2]));
        } else {
          *reinterpret_cast<float4*>(a.part_o + (slot * a.gs + head) * HD + f) = s;
          if (f == 0) *reinterpret_cast<float4*>(a.part_s + (slot * a.gs + head) * 4) = make_float4(fin_s[head][0], fin_s[head][1], fin_s[head][2], 0.f);
        }
      }
    }
    if (!more) break;
    __syncthreads();                           // shared memory is the next piece's
    p = next;
  }
  if constexpr (CLUSTER) {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    const int rank = (int)cl.block_rank();
    for (int e = rank * DA_THREADS + threadIdx.x; e < a.gs * (HD / 4); e += a.cluster * DA_THREADS) {
      const int head = e / (HD / 4), f = e % (HD / 4) * 4;
      DaJoin j;
      j.none();
      for (int r = 0; r < a.cluster; r++) {
        const float* st = cl.map_shared_rank(&fin_s[head][0], r);
        j.add(st[0], st[1], st[2], *reinterpret_cast<const float4*>(cl.map_shared_rank(res_s + head * HD + f, r)));
      }
      da_store(a.out + (long long)p.t * a.ldo + (long long)(p.kvh * a.gs + head) * HD + f, j.s, j.inverse());
    }
    cl.sync();                                 // (nobody leaves whose shared memory is read)
  }
  if (dead)
    for (int i = 0; i < 1000; i++) __nanosleep(1000);          // copies on their way land in what is still this CTA's
}

// The pieces of pairs that several CTAs of the launch before (of n_ctas) had: a block to ``heads`` of a pair's heads (a power of two), whose threads'
// groups have every so many'th piece of one each.  (One token of 100,001 keys has 74 pieces to a pair: one after the other in a block to a pair
// they took 25 us.  64 tokens of 28 heads in blocks to a head each: 1,792, twice what fits beside the launch before and finds out what it
// has to join meanwhile, 10 us; ``heads`` is as many as bring the blocks to four a multiprocessor.)
template <int HD, int THREADS>
__global__ void __launch_bounds__(THREADS) decode_fp8_join_kernel(const DaArgs a, int n_ctas, int heads) {
  constexpr int LANES = HD / 4;
  __shared__ int sums[DA_TOKENS + 1], scratch[THREADS / 32];
  __shared__ DaJoin got[THREADS];
  pdl_launch_dependents();
  const DaList list = da_list<THREADS>(a, sums, scratch);
  const int sets = (a.gs + heads - 1) / heads, pair = blockIdx.x / sets, t = pair / a.pages.G, kvh = pair % a.pages.G, per = list.units_of(t);
  const long long U = (long long)list.all() * a.pages.G;
  n_ctas = da_taking(U, n_ctas, a.T * a.pages.G, list.most);
  const int from = list.units_before(t) * a.pages.G + kvh * per;
  const int2 cut = da_cut_by(U, n_ctas, from, per);
  const int c0 = cut.x, c1 = cut.y;
  // whether CTA c0 has something before this pair: then this is its second piece
  bool second = false;
  if (c0 < c1) {
    const int at = da_cut(U, n_ctas, c0);
    if (at < from) {
      const int u = list.token(at, a.pages.G), of = list.units_of(u);
      second = da_snap(at, (at - list.units_before(u) * a.pages.G) % of, of) < from;
    }
  }
  pdl_wait();                                  // (also where there is nothing to join: the next launch waits for this one alone)
  if (c0 >= c1) return;
  const int f = threadIdx.x % LANES * 4, slot = threadIdx.x / LANES, h = blockIdx.x % sets * heads + (slot & (heads - 1));
  const int group = slot / heads, groups = THREADS / LANES / heads;
  DaJoin j;
  j.none();
  if (h < a.gs) {
#pragma unroll 4
    for (int i = c0 + group; i <= c1; i += groups) {
      const long long at = (2ll * i + (i == c0 && second ? 1 : 0)) * a.gs + h;
      const float4 st = __ldcg(reinterpret_cast<const float4*>(a.part_s + at * 4));
      j.add(st.x, st.y, st.z, __ldcg(reinterpret_cast<const float4*>(a.part_o + at * HD + f)));
    }
  }
  got[threadIdx.x] = j;
  __syncthreads();
  if (group || h >= a.gs) return;
  for (int i = 1; i < groups && c0 + i <= c1; i++) {
    const DaJoin& k = got[i * heads * LANES + threadIdx.x];
    j.add(k.sum, k.mz, k.mw, k.s);
  }
  da_store(a.out + (long long)t * a.ldo + (long long)(kvh * a.gs + h) * HD + f, j.s, j.inverse());
}

// the number of the first wait that ran out (made with the module, not by the first call, which may be a captured one)
static __device__ int da_status;
static int* da_status_word() {
  static int* words[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  if (!words[dev]) {
    void* w = nullptr;
    if (cudaGetSymbolAddress(&w, da_status) != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    words[dev] = (int*)w;
  }
  return words[dev];
}

// How a launch over T tokens of up to max_keys keys is cut: CTAs, and how many of them are a pair's cluster (0: units are dealt out).  A cluster costs 5 us
// and 0.85 for each of its CTAs' units, however short the other tokens are; dealing out costs 13 and more with the tokens (a list of them in every CTA,
// pieces, the launch that joins them), and takes no longer for one long token among short ones.  With 28 + 4 heads, dealt out and in clusters: 1 token of
// 12,000 keys 14.3 and 11.2 us, of 24,000 15.4 and 16.3; 8 of 500 8.1 and 6.6, of up to 4,000 13.6 and 12.9; 16 of up to 4,000 16.0 and 18.4; 32 of 1,000
// 17.7 and 11.3, of up to 4,000 22.2 and 30.7; 64 of up to 300 12.2 and 8.8, of up to 2,000 23.1 and 23.3, of up to 8,000 55.6 and 76.2; 256 of up to 500
// 34.5 and 30.5, of up to 2,000 64.1 and 64.4.
struct DaPlan { int ctas, cluster; };
static DaPlan da_plan(int T, int G, int gs, int window, int max_keys, int sms) {
  const long long keys = window > 0 && window < max_keys ? window + 15ll : max_keys;
  const long long per = (keys + DA_UNIT - 1) / DA_UNIT, pairs = (long long)T * G, at_a_time = (long long)(gs > 8 ? 1 : 2) * sms;
  // a CTA to a multiprocessor, at most
  int n = 1;
  while (n < DA_MAX_CLUSTER && n < per && 2 * n * pairs <= sms) n *= 2;
  if (per <= (pairs > sms ? 16 : 8) * n && n * pairs <= 0x7fffffffll) return {(int)(n * pairs), n};
  return {(int)(pairs * per < at_a_time ? pairs * per : at_a_time), 0};
}

// float32 numbers of scratch memory that a call takes: the most that a round of it does.  Rounds are DA_TOKENS and what is left, each with a plan of its own:
// the rest may be dealt out where a full round goes in clusters
extern "C" long long qd_decode_attention_fp8_scratch(int T, int H, int G, int d, int window, int max_keys, int sms) {
  if (T < 1 || G < 1 || H < 1) return 0;
  long long most = 0;
  for (const int n : {T < DA_TOKENS ? T : DA_TOKENS, T % DA_TOKENS}) {
    if (!n) continue;
    const DaPlan plan = da_plan(n, G, H / G, window, max_keys, sms);
    const long long floats = plan.cluster ? 0 : 2ll * plan.ctas * (H / G) * (d + 4);
    if (floats > most) most = floats;
  }
  return most;
}
// and the kernels that it launches: a round's, and where that is dealt out the one that joins its pieces
extern "C" int qd_decode_attention_fp8_launches(int T, int H, int G, int window, int max_keys, int sms) {
  if (T < 1 || G < 1 || H < 1) return 0;
  auto of_round = [&](int n) { return da_plan(n, G, H / G, window, max_keys, sms).cluster ? 1 : 2; };
  return (T >= DA_TOKENS ? T / DA_TOKENS * of_round(DA_TOKENS) : 0) + (T % DA_TOKENS ? of_round(T % DA_TOKENS) : 0);
}

template <int HD, int NT, bool CLUSTER>
static int da_launch(const CUtensorMap& map, const DaArgs& a, int ctas, int sms, cudaStream_t stream) {
  const int smem = 1024 + DA_WARPS * (DA_STAGES * 32 * HD + 8 * 8 * (HD / 8 + 4) * 4);
  auto kernel = decode_fp8_kernel<HD, NT, CLUSTER>;
  static bool allowed[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return QD_ERR_UNSUPPORTED;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        (CLUSTER && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)) {
      cudaGetLastError();
      return QD_ERR_UNSUPPORTED;
    }
    allowed[dev] = true;
  }
  if (!CLUSTER) {
    qd_launch(kernel, dim3(ctas), dim3(DA_THREADS), smem, stream, map, a);
    int heads = 1;
    while (heads < 8 && heads < a.gs && (long long)a.T * a.pages.G * ((a.gs + heads - 1) / heads) > 4ll * sms) heads *= 2;
    // few blocks have many threads, for as many pieces at a time (one token, 28 + 4 heads, 24,000 keys 14.7 us, with 256 threads 16.1, 100,000 26.2 and 27.9;
    // two of 32,000 19.9 and 19.0: past some thirty blocks the wait for room beside the launch before is longer)
    const dim3 blocks(a.T * a.pages.G * ((a.gs + heads - 1) / heads));
    if (4 * (int)blocks.x <= sms) qd_launch(decode_fp8_join_kernel<HD, 1024>, blocks, dim3(1024), 0, stream, a, ctas, heads);
    else qd_launch(decode_fp8_join_kernel<HD, DA_THREADS>, blocks, dim3(DA_THREADS), 0, stream, a, ctas, heads);
    return qd_last_error();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(DA_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = qd_pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, map, a);
  return qd_last_error();
}
template <int HD>
static int da_launch_of(const CUtensorMap& map, const DaArgs& a, int ctas, int sms, cudaStream_t stream) {
  if (a.cluster) return a.gs <= 8 ? da_launch<HD, 1, true>(map, a, ctas, sms, stream) : da_launch<HD, 2, true>(map, a, ctas, sms, stream);
  return a.gs <= 8 ? da_launch<HD, 1, false>(map, a, ctas, sms, stream) : da_launch<HD, 2, false>(map, a, ctas, sms, stream);
}

// q, out: bfloat16 rows [T, H d], ``ldq`` and ``ldo`` apart; table [table_rows, max_blocks] of pages of ps tokens (a multiple of 16), its row of token t is
// token_req[t]; the token sees the keys up to positions[t] (none below zero), the last ``window`` of them if that is positive.  No position may be
// beyond max_keys - 1 (later keys are not seen).  scratch: qd_decode_attention_fp8_scratch of the same sizes, on 16 bytes; null where that is 0.
extern "C" int qd_decode_attention_fp8(const void* q, long long ldq, void* out, long long ldo, const void* pages, long long n_pages, const int* table,
                                       int max_blocks, int table_rows, const int* token_req, const int* positions, int T, int H, int G, int d, int ps,
                                       float scale, int window, int max_keys, float* scratch, int sms, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (G < 1 || H < 1 || H % G || H / G > 16 || (d != 64 && d != 128) || ps < 16 || ps % 16 || n_pages < 1 || n_pages > 0x7fffffffll || max_blocks < 1 ||
      table_rows < 1 || max_keys < 1 || window < 0 || (long long)max_blocks * ps < max_keys)
    return QD_ERR_UNSUPPORTED;
  if ((((uintptr_t)q | (uintptr_t)out | (uintptr_t)pages) & 15) || ldq % 8 || ldo % 8) return QD_ERR_UNSUPPORTED;
  const int gs = H / G;
  if (!scratch && qd_decode_attention_fp8_scratch(T, H, G, d, window, max_keys, sms)) return QD_ERR_UNSUPPORTED;
  // the units of a launch fit 31 bits
  if ((long long)(T < DA_TOKENS ? T : DA_TOKENS) * G * (max_keys / DA_UNIT + 2 + DA_PIECE) > 0x7fffffffll) return QD_ERR_UNSUPPORTED;
  int* status = da_status_word();
  CUtensorMap map;
  if (!status || !c8_make_map(&map, pages, n_pages, G, ps, d)) return QD_ERR_UNSUPPORTED;
  for (int t = 0; t < T; t += DA_TOKENS) {
    const int n = T - t < DA_TOKENS ? T - t : DA_TOKENS;
    const DaPlan plan = da_plan(n, G, gs, window, max_keys, sms);
    const DaArgs a = {(const bf16*)q + t * ldq, ldq, (bf16*)out + t * ldo, ldo, {(unsigned char*)pages, c8_page_bytes(G, ps, d), G, ps, d}, (int)n_pages,
                      table, max_blocks, table_rows, token_req + t, positions + t, n, H, gs, window, max_keys, scale * 1.4426950408889634f,
                      scratch, scratch + 2ll * plan.ctas * gs * d, plan.cluster, ps & (ps - 1) ? -1 : __builtin_ctz(ps), status};
    const int rc = d == 128 ? da_launch_of<128>(map, a, plan.ctas, sms, stream) : da_launch_of<64>(map, a, plan.ctas, sms, stream);
    if (rc) return rc;
  }
  return 0;
}

QD_DEFINE_WAIT_PROBE(qd_decode_attention_fp8_wait_probe, tc_wait(bar, 0, dead, 0, poll_limit), da_status_word, 99)

// 0 if no kernel of this library has recorded a wait that ran out on the current device.  Synchronises.
extern "C" int qd_decode_attention_fp8_status() {
  int* status = da_status_word();
  if (!status) return -1;
  int v = 0;
  if (cudaMemcpy(&v, status, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) return -1;
  if (v) cudaMemset(status, 0, sizeof(int));
  return v;
}
