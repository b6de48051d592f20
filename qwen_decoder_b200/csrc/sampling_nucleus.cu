// A token of each row of logits by temperature, top-k, top-p and min-p, from a given number r in [0, 1):
//
//   w_i = e^((z_i - max z) / T),   K = {z_i >= the k-th largest},   N = {z_i >= t}: t the largest logit with
//   sum_{K, z_i >= t} w_i >= top_p sum_K w_i,   M = {w_i >= min_p};   the first i of K, N and M whose running sum of w reaches r times all of it
//
// (logits that are equal are in or out together).  Temperature 0 is the largest logit, of equal ones the first.  The reference has
// temperature and top-k (common.cpp:576-629).
//
// Which token a number falls to, and which logit is the last of a nucleus, changes where sums are next to a border, and rows have a hundred
// thousand borders.  So weights are whole numbers, w 2^44 to within three (2^40 for rows of more than 2^18 logits): their sums are exact, in whatever
// order, and a row's token does not depend on how its work is shared.  What is lost is 3 2^-44 of the largest weight for each at most.
//
// A cluster of S CTAs shares a row, contiguous parts of it (in shared memory where they fit).  The k-th largest logit and t are found
// alike, by histograms (counts, or counts and weights) over the cluster: first over 1,472 equal steps of z below the maximum, down to 46 ln 2 T,
// where weights end (the logits of a row are spread over many of these, so that few additions meet; in steps of the number's leading bits
// they would not be); then the logits of the step that the border lies in go to one CTA, which puts them in order.  Where they are more than
// SN_NEAR (a thousand equal logits), histograms over steps of the logit's bits follow, until a step is one number.
// Bound by the row's reading for the rest and by the trips over the cluster, two to a histogram.
//
// A top-k of up to 256 needs none of that: the k-th largest of a CTA's threads' own maxima has k logits that reach it, as the least of the
// CTAs' ceil(k / S)-th ones has; what reaches the larger of these bounds is little more than k logits, which go to one CTA's list, are put in order
// there and decide the rest.
#include "common.cuh"
#include <cooperative_groups.h>
#include <math.h>

namespace cg = cooperative_groups;

#define SN_THREADS 512
#define SN_WARPS (SN_THREADS / 32)
#define SN_BINS 2048
#define SN_EACH (SN_BINS / SN_THREADS)
#define SN_MAX_SHARES 16
#define SN_KEEP 36864                            // logits that a CTA holds in shared memory
#define SN_POWERS 4096                           // to an octave
#define SN_OCTAVES 46                            // below the maximum a weight is 0
#define SN_STEP 7                                // log2 of the powers to a step of the first histogram
static_assert((SN_OCTAVES * SN_POWERS >> SN_STEP) + 1 < SN_BINS, "steps of the first histogram");
#define SN_FEW 256                               // a top-k up to here goes by the list
#define SN_LIST 2048
#define SN_AHEAD 4                               // 16 bytes each that a thread has on their way
#define SN_NEAR 1024                             // logits next to a border that are put in order

struct SnArgs {
  const float* logits;
  long long ld;
  const float *temperature, *top_p, *min_p, *draws;
  const int* top_k;
  int* out;
  int V, shares, vec, keep, weights, bits, only;          // keep, weights: a CTA's logits and their weights are in shared memory
};
// 2^(-k / 4096) over 2^44: powers of the twelfth root of a half, each root the whole root of the one before, over 2^63
struct SnPowers {
  unsigned long long of[SN_POWERS];
  static constexpr unsigned long long root(unsigned __int128 v) {            // whole part, bit by bit
    unsigned long long r = 0;
    for (int b = 63; b >= 0; b--) {
      const unsigned long long t = r | 1ull << b;
      if ((unsigned __int128)t * t <= v) r = t;
    }
    return r;
  }
  constexpr SnPowers() : of() {
    unsigned long long s = 1ull << 62, p = 1ull << 63;
    for (int i = 0; i < 12; i++) s = root((unsigned __int128)s << 63);
    for (int k = 0; k < SN_POWERS; k++) {
      of[k] = (p + (1 << 18)) >> 19;
      p = (unsigned long long)((unsigned __int128)p * s >> 63);
    }
  }
};
__device__ const __align__(16) SnPowers sn_powers = SnPowers();

struct SnShared {
  union {
    struct {
      uint2 mine[SN_BINS];                       // a 64-bit sum each, the low half in x
      unsigned long long all[SN_BINS];           // of the cluster
    };
    struct {                                     // with a small top-k, of the cluster's first CTA: logits as keys above the complement of their
      unsigned long long list[SN_LIST], mass[SN_LIST];       // index, the largest first; sums of weights up to each
    };
  };
  __align__(16) unsigned long long powers[SN_POWERS];
  unsigned long long near[SN_NEAR];              // of the cluster's first CTA: keys
  int listed;
  unsigned long long got[2][SN_MAX_SHARES];      // a word of each CTA
  unsigned long long warps[SN_WARPS], above;
  unsigned bin, ends[2], key, last_step[2], counts[SN_WARPS];
};

__device__ __forceinline__ unsigned sn_order(float z) {             // ascending; no number: 0
  const unsigned u = __float_as_uint(z + 0.0f);                      // (both zeros alike)
  return z != z ? 0u : u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float sn_value(unsigned order) { return __uint_as_float(order ^ (order >> 31 ? 0x80000000u : 0xffffffffu)); }
#define SN_LOWEST 0x00800000u                                        // the order of the lowest number: minus infinity lies below

struct SnRow {
  const float* z;                                // of this CTA's part, in shared memory or the row itself
  int n, vec, warp_from, warp_to;                // how many, 16 bytes at a time; of this warp
  float top;                                     // the maximum
  float c, c2;                                   // 1 / (T log 2)
  int bits;
  const unsigned long long* powers;              // in shared memory
  unsigned long long* weight;                    // of this CTA's part, where they are kept (else null)
};
// four neighbouring logits, minus infinity behind the end
__device__ __forceinline__ void sn_four(const SnRow& r, int i, float (&v)[4]) {
  if (r.vec && i + 4 <= r.n) {
    const float4 f = *reinterpret_cast<const float4*>(r.z + i);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = i + j < r.n ? r.z[i + j] : -INFINITY;
  }
}
// y = (max - z) / (T log 2) in 4,096ths, of which the first histogram's steps are 128; SN_OCTAVES of them, and what is no number, are far
__device__ __forceinline__ int sn_place(const SnRow& r, float z) {
  const float p = (r.top - z) * r.c;
  return p < SN_OCTAVES ? __float_as_int(fmaf(p, (float)SN_POWERS, 12582912.f)) - 0x4b400000 : SN_OCTAVES * SN_POWERS;
}
__device__ __forceinline__ unsigned sn_step(const SnRow& r, float z) { return (unsigned)sn_place(r, z) >> SN_STEP; }
// e^((z - max) / T) over 2^-44 (2^-bits) as a whole number, within three of it (2.6 of 6 million, without a bias), in 32-bit arithmetic (an instruction of 64-bit floating point is some
// 20 cycles of a scheduler).  With d = max - z and c = 1 / (T log 2), each a sum of two float32 numbers, y = c d is one to 2^-47 of itself; with
// ``place`` k of it taken away x / log 2 is left, and the result is 2^(-k / 4096) (1 - x + x^2 / 2 - x^3 / 6), |x| < 2^-13.
__device__ __forceinline__ unsigned long long sn_weight(const SnRow& r, float z, int k) {
  const float d = r.top - z, back = d - r.top, d2 = (r.top - (d - back)) - (z + back);       // (what the difference lost)
  const float p = d * r.c;
  const float e = fmaf(d2, r.c, fmaf(d, r.c2, fmaf(d, r.c, -p)));
  const float f = fmaf((float)k, -1.f / SN_POWERS, p), y = f + e, y2 = e - (y - f);
  const float x = y * 0.693147182f, x2 = fmaf(y2, 0.693147182f, fmaf(y, -1.90465421e-9f, fmaf(y, 0.693147182f, -x)));
  const float rest = fmaf(x * x, fmaf(x, 1.f / 6, -0.5f), x2);
  const int less = __float2int_rn(x * 17592186044416.f) + (__float_as_int(fmaf(rest, 17592186044416.f, 12582912.f)) - 0x4b400000);       // over 2^-44
  const unsigned long long w = r.powers[k & (SN_POWERS - 1)];
  const unsigned long long whole = w - (long long)(int)(((long long)(int)(w >> 14) * less + (1 << 29)) >> 30);
  const int down = 44 - r.bits + (k / SN_POWERS);
  return k < SN_OCTAVES * SN_POWERS ? whole + (1ull << down >> 1) >> down : 0ull;
}
// (one copy of the code for what is asked for seldom: a launch goes through most of its code once, and waits for it where it is long)
__device__ __noinline__ unsigned long long sn_weight_once(const SnRow& r, float z) { return sn_weight(r, z, sn_place(r, z)); }
// of this CTA's four logits from i on, z; none of those below ``least``
__device__ __forceinline__ void sn_weights_at(const SnRow& r, int i, const float (&z)[4], float least, unsigned long long (&w)[4]) {
  if (r.weight) {
    const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(r.weight + i), b = *reinterpret_cast<const ulonglong2*>(r.weight + i + 2);
    w[0] = a.x; w[1] = a.y; w[2] = b.x; w[3] = b.y;
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = z[j] >= least ? w[j] : 0;
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = z[j] >= least ? sn_weight_once(r, z[j]) : 0;
  }
}
// the least weight that min_p leaves
__device__ __forceinline__ unsigned long long sn_least(const SnRow& r, float min_p) {
  return (unsigned long long)ceil(fmin((double)min_p, 1.0) * (double)(1ull << r.bits));
}

// every CTA's word, in every CTA.  Calls in turn use two places, so that a fast CTA's next word does not meet a slow one's reading.
__device__ __forceinline__ const unsigned long long* sn_exchange(SnShared& s, int shares, unsigned long long word, int& turn) {
  unsigned long long* all = s.got[turn];
  if (shares == 1) {
    if (threadIdx.x == 0) all[0] = word;
    __syncthreads();
  } else {
    cg::cluster_group cl = cg::this_cluster();
    if (threadIdx.x < shares) cl.map_shared_rank(all, threadIdx.x)[cl.block_rank()] = word;
    cl.sync();
  }
  turn ^= 1;
  return all;
}
// a word of every warp, in every thread: op over the block
template <typename Op>
__device__ __forceinline__ unsigned long long sn_block(SnShared& s, unsigned long long v, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.warps[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s.warps[0];
#pragma unroll
  for (int w = 1; w < SN_WARPS; w++) v = op(v, s.warps[w]);
  return v;
}
// The first key for which ``holds``, which is false up to some key, at lo among them, and true from there on, at hi among them.  A whole warp.
template <typename F>
__device__ __forceinline__ unsigned sn_first_key(unsigned lo, unsigned hi, F holds) {
  const unsigned lane = threadIdx.x & 31;
  while (hi - lo > 1) {
    const unsigned long long span = hi - lo;
    const unsigned at = lo + (unsigned)(span * (lane + 1) / 33);
    const unsigned yes = __ballot_sync(0xffffffffu, at > lo && holds(at));
    const unsigned first = yes ? __ffs(yes) - 1 : 32;
    if (first < 32) hi = lo + (unsigned)(span * (first + 1) / 33);
    if (first > 0) lo = lo + (unsigned)(span * first / 33);
  }
  return hi;
}

// n 64-bit numbers in order, the largest first, in room for the next power of two.  Up to 384 by counting for each how many come before it (200:
// 2,000 cycles), more by bitonic steps (36 of them for 200, 150 cycles each with the barrier).
__device__ void sn_sort(unsigned long long* list, int n) {
  if (n <= 384) {
    __syncthreads();
    const unsigned long long own = (int)threadIdx.x < n ? list[threadIdx.x] : 0;
    int before = 0;
#pragma unroll 4
    for (int i = 0; i < n; i++) before += list[i] > own || list[i] == own && i < (int)threadIdx.x;
    __syncthreads();
    if ((int)threadIdx.x < n) list[before] = own;
    __syncthreads();
    return;
  }
  int size = 32;
  while (size < n) size *= 2;
  for (int i = n + threadIdx.x; i < size; i += SN_THREADS) list[i] = 0;
  for (int span = 2; span <= size; span *= 2)
    for (int step = span / 2; step > 0; step /= 2) {
      __syncthreads();
      for (int i = threadIdx.x; i < size / 2; i += SN_THREADS) {
        const int x = 2 * i - (i & (step - 1)), y = x + step;
        const unsigned long long p = list[x], q = list[y];
        if ((p < q) == !(x & span)) { list[x] = q; list[y] = p; }
      }
    }
  __syncthreads();
}
// sums up to each of n words, by the whole block; all of them
template <typename F>
__device__ unsigned long long sn_sums(SnShared& s, int n, F word) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long carry = 0;
  for (int i0 = 0; i0 < n; i0 += SN_THREADS) {
    const int i = i0 + threadIdx.x;
    unsigned long long sum = i < n ? word(i) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) s.warps[warp] = sum;
    __syncthreads();
    unsigned long long ahead = carry;
    for (int w = 0; w < SN_WARPS; w++) {
      if (w < warp) ahead += s.warps[w];
      carry += s.warps[w];
    }
    if (i < n) s.mass[i] = ahead + sum;
    __syncthreads();
  }
  return carry;
}
// The border among the n keys of ``near``, above all of which lies ``above``.
template <bool MASS>
__device__ unsigned sn_among(SnShared& s, const SnRow& r, int n, unsigned long long above, double want) {
  sn_sort(s.near, n);
  sn_sums(s, n, [&](int i) { return MASS ? sn_weight_once(r, sn_value((unsigned)s.near[i])) : 1ull; });
  if (threadIdx.x == 0) s.bin = n - 1;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += SN_THREADS)
    if ((double)(above + s.mass[i]) >= want && (i == 0 || !((double)(above + s.mass[i - 1]) >= want))) s.bin = i;
  __syncthreads();
  return (unsigned)s.near[s.bin];
}

// The largest key t so that the logits of keys from t on, none below ``floor`` among them, hold ``want`` or more: counts, or of weights the
// share ``want`` of them all.  ``floor`` where there is less than that down to where weights end.
template <bool MASS>
__device__ unsigned sn_border(SnShared& s, const SnRow& r, int shares, unsigned floor, double want) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned top = sn_order(r.top);
  unsigned k_lo = floor, k_hi = top;             // the border is one of these
  unsigned long long above = 0;                  // what lies above them
  for (int level = 0;; level++) {
    int shift = 0;
    while (((k_hi - k_lo) >> shift) >= SN_BINS) shift++;
    for (int b = threadIdx.x; b < SN_BINS; b += SN_THREADS) s.mine[b] = make_uint2(0, 0);
    __syncthreads();
    const float from_z = sn_value(k_lo), to_z = sn_value(k_hi);
#pragma unroll 1
    for (int i = r.warp_from + 4 * lane; i < r.warp_to; i += 128) {
      float v[4];
      unsigned bin[4];
      unsigned long long w[4] = {1, 1, 1, 1};
      sn_four(r, i, v);
      if (level == 0) {
        int k[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          k[j] = v[j] >= from_z ? sn_place(r, v[j]) : SN_OCTAVES * SN_POWERS;
          bin[j] = k[j] < SN_OCTAVES * SN_POWERS ? (unsigned)k[j] >> SN_STEP : SN_BINS;
        }
        if (MASS) {
#pragma unroll
          for (int j = 0; j < 4; j++) w[j] = sn_weight(r, v[j], k[j]);
          if (r.weight) {
            *reinterpret_cast<ulonglong2*>(r.weight + i) = make_ulonglong2(w[0], w[1]);
            *reinterpret_cast<ulonglong2*>(r.weight + i + 2) = make_ulonglong2(w[2], w[3]);
          }
        }
      } else {
        bool any = false;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          bin[j] = v[j] >= from_z && v[j] <= to_z ? (k_hi - sn_order(v[j])) >> shift : SN_BINS;
          any |= bin[j] < SN_BINS;
        }
        if (MASS && any) sn_weights_at(r, i, v, from_z, w);
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (bin[j] < SN_BINS) {
          const unsigned lo = (unsigned)w[j], old = atomicAdd(&s.mine[bin[j]].x, lo);
          if (MASS) {
            const unsigned hi = (unsigned)(w[j] >> 32) + (old > 0xffffffffu - lo ? 1u : 0u);
            if (hi) atomicAdd(&s.mine[bin[j]].y, hi);
          }
        }
    }
    if (shares > 1) {
      // a CTA adds up its part of the steps: as many neighbouring threads as CTAs read one's sums each, all of theirs before the first is stored, and
      // hand the whole to one each
      cg::cluster_group cl = cg::this_cluster();
      cl.sync();
      const int per = SN_BINS / shares, b0 = (int)cl.block_rank() * per, c = threadIdx.x % shares, step = SN_THREADS / shares;
      const uint2* from = cl.map_shared_rank(s.mine, c) + b0 + threadIdx.x / shares;
      unsigned long long* to = cl.map_shared_rank(s.all, c) + b0 + threadIdx.x / shares;
      uint2 got[SN_EACH];                        // (SN_BINS / shares of them, SN_THREADS / shares at a time)
#pragma unroll
      for (int u = 0; u < SN_EACH; u++) got[u] = from[u * step];
#pragma unroll
      for (int u = 0; u < SN_EACH; u++) {
        unsigned long long sum = ((unsigned long long)got[u].y << 32) + got[u].x;
        for (int o = shares / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        to[u * step] = sum;
      }
      cl.sync();
    } else {
      __syncthreads();
      for (int b = threadIdx.x; b < SN_BINS; b += SN_THREADS) s.all[b] = ((unsigned long long)s.mine[b].y << 32) + s.mine[b].x;
      __syncthreads();
    }
    // the first step with which the sum from above reaches what is wanted
    unsigned long long own[SN_EACH], sum = 0;
#pragma unroll
    for (int u = 0; u < SN_EACH; u++) { own[u] = s.all[threadIdx.x * SN_EACH + u]; sum += own[u]; }
    unsigned long long incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) s.warps[warp] = incl;
    if (threadIdx.x == 0) s.bin = SN_BINS;
    __syncthreads();
    unsigned long long run = above + incl - sum, total = 0;
#pragma unroll
    for (int w = 0; w < SN_WARPS; w++) {
      run += w < warp ? s.warps[w] : 0;
      total += s.warps[w];
    }
    if (MASS && level == 0) want = fmax(want * (double)total, 1.0);
    if (!((double)run >= want) && (double)(run + sum) >= want) {
      int u = 0;
      while (u < SN_EACH - 1 && !((double)(run + own[u]) >= want)) run += own[u++];
      s.bin = threadIdx.x * SN_EACH + u;
      s.above = run;
    }
    __syncthreads();
    const unsigned bin = s.bin;
    if (bin >= SN_BINS) return floor;
    above = s.above;
    if (level == 0) {
      // the step's logits to the first CTA, in any order
      int* count = shares > 1 ? cg::this_cluster().map_shared_rank(&s.listed, 0) : &s.listed;
      unsigned long long* near = shares > 1 ? cg::this_cluster().map_shared_rank(s.near, 0) : s.near;
#pragma unroll 1
      for (int i = r.warp_from + 4 * lane; i < r.warp_to; i += 128) {
        float v[4];
        sn_four(r, i, v);
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (v[j] >= from_z && v[j] <= to_z && sn_step(r, v[j]) == bin) {
            const int at = atomicAdd(count, 1);
            if (at < SN_NEAR) near[at] = sn_order(v[j]);
          }
      }
      if (shares > 1) cg::this_cluster().sync();
      else __syncthreads();
      const int n = *count;
      if (n <= SN_NEAR && (shares == 1 || cg::this_cluster().block_rank() == 0)) {
        const unsigned key = sn_among<MASS>(s, r, n, above, want);
        if ((int)threadIdx.x < shares) *(shares > 1 ? cg::this_cluster().map_shared_rank(&s.key, threadIdx.x) : &s.key) = key;
        __syncthreads();
      }
      if (shares > 1) cg::this_cluster().sync();           // (the first CTA's list has been counted, too)
      else __syncthreads();
      if (threadIdx.x == 0) s.listed = 0;
      if (n <= SN_NEAR) return s.key;
    }
    if (level) {
      k_hi -= bin << shift;
      if (!shift) return k_hi;
      const unsigned wide = (1u << shift) - 1;
      k_lo = k_hi - k_lo > wide ? k_hi - wide : k_lo;
    } else {
      // the keys of this step of z, by bisection of the very expression: the first of the step, the first behind it
      if (warp < 2) {
        const unsigned end = sn_first_key(k_lo - 1, top + 1, [&](unsigned key) {
          return key > top || (warp ? sn_step(r, sn_value(key)) < bin : sn_step(r, sn_value(key)) <= bin);
        });
        if (lane == 0) s.ends[warp] = end;
      }
      __syncthreads();
      k_lo = s.ends[0];
      k_hi = s.ends[1] - 1;
    }
    if (k_lo == k_hi) return k_hi;
    __syncthreads();                             // shared memory is the next histogram's
  }
}

// A token by the list of a small top-k, or -1 where more logits reach the bound than it holds.  ``best``: this thread's maximum.  The cluster's first CTA
// knows the token, the others -1 or 0.
__device__ int sn_by_list(SnShared& s, const SnRow& r, int shares, int rank, int first, int k, unsigned best, float top_p, float min_p, float draw,
                          int likeliest, int& turn) {
  const int lane = threadIdx.x & 31;
  // the bound: of the threads' maxima the least of those in the steps between the row's maximum and the least of them that hold k, or ceil(k / S)
  unsigned* steps = reinterpret_cast<unsigned*>(s.list);
  const int warp = threadIdx.x >> 5, of_all = (k + shares - 1) / shares;
  const unsigned lowest = (unsigned)sn_block(s, best ? best : 0xffffffffu, [](unsigned long long x, unsigned long long y) { return x < y ? x : y; });
  for (int i = threadIdx.x; i < SN_BINS; i += SN_THREADS) steps[i] = 0;
  __syncthreads();
  const float scale = (float)(SN_BINS - 2) / fmaxf(r.top - sn_value(lowest), 1e-30f);
  const unsigned own = best ? (unsigned)fminf((r.top - sn_value(best)) * scale, (float)(SN_BINS - 2)) : SN_BINS - 1;      // (the last: no number)
  atomicAdd(&steps[own], 1u);
  __syncthreads();
  unsigned held[SN_EACH], sum = 0;
#pragma unroll
  for (int u = 0; u < SN_EACH; u++) { held[u] = steps[threadIdx.x * SN_EACH + u]; sum += held[u]; }
  unsigned upto = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) s.counts[warp] = upto;
  __syncthreads();
  int before = (int)(upto - sum);
#pragma unroll
  for (int w = 0; w < SN_WARPS; w++) before += w < warp ? s.counts[w] : 0;
#pragma unroll
  for (int u = 0; u < SN_EACH; u++) {
    if (before < k && k <= before + (int)held[u]) s.last_step[0] = threadIdx.x * SN_EACH + u;
    if (before < of_all && of_all <= before + (int)held[u]) s.last_step[1] = threadIdx.x * SN_EACH + u;
    before += held[u];
  }
  if (threadIdx.x < 2) s.ends[threadIdx.x] = 0xffffffffu;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const unsigned mine = __reduce_min_sync(0xffffffffu, own <= s.last_step[e] ? best : 0xffffffffu);
    if (lane == 0) atomicMin(&s.ends[e], mine);
  }
  __syncthreads();
  const unsigned long long* words = sn_exchange(s, shares, (unsigned long long)s.ends[0] << 32 | s.ends[1], turn);
  unsigned most = 0, least = 0xffffffffu;
  for (int c = 0; c < shares; c++) {
    most = max(most, (unsigned)(words[c] >> 32));
    least = min(least, (unsigned)words[c]);
  }
  const unsigned bound = max(max(most, least), SN_LOWEST);
  // what reaches it, to the first CTA's list (in any order)
  cg::cluster_group cl = cg::this_cluster();
  int* count = shares > 1 ? cl.map_shared_rank(&s.listed, 0) : &s.listed;
  unsigned long long* list = shares > 1 ? cl.map_shared_rank(s.list, 0) : s.list;
  const float bound_z = sn_value(bound);
  for (int i0 = r.warp_from + 4 * lane; i0 < r.warp_to; i0 += 128 * SN_AHEAD) {
    float v[SN_AHEAD][4];
#pragma unroll
    for (int u = 0; u < SN_AHEAD; u++) {
      v[u][0] = v[u][1] = v[u][2] = v[u][3] = -INFINITY;
      if (i0 + 128 * u < r.warp_to) sn_four(r, i0 + 128 * u, v[u]);
    }
#pragma unroll
    for (int u = 0; u < SN_AHEAD; u++)
      if (fmaxf(fmaxf(v[u][0], v[u][1]), fmaxf(v[u][2], v[u][3])) >= bound_z) {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (v[u][j] >= bound_z) {
            const int at = atomicAdd(count, 1);
            if (at < SN_LIST) list[at] = (unsigned long long)sn_order(v[u][j]) << 32 | (0xffffffffu - (unsigned)(first + i0 + 128 * u + j));
          }
      }
  }
  if (shares > 1) cl.sync();
  else __syncthreads();
  const int n = *count;
  if (n > SN_LIST) {
    if (shares > 1) cl.sync();                   // (nobody's shared memory becomes something else while it is read)
    else __syncthreads();
    if (threadIdx.x == 0) s.listed = 0;
    return -1;
  }
  if (shares > 1) cl.sync();
  if (threadIdx.x == 0) s.listed = 0;
  if (rank) return 0;
  sn_sort(s.list, n);
  // the k-th largest and its equals, sums of weights
  auto key_at = [&](int i) { return (unsigned)(s.list[i] >> 32); };
  const unsigned kth = key_at(min(k, n) - 1);
  const unsigned long long carry = sn_sums(s, n, [&](int i) { return key_at(i) >= kth ? sn_weight_once(r, sn_value(key_at(i))) : 0ull; });
  // the last key that stays: the k-th largest, or of the nucleus, or of those with enough probability
  if (threadIdx.x == 0) { s.ends[0] = kth; s.key = 0xffffffffu; s.ends[1] = kth; }
  __syncthreads();
  const double want = top_p < 1.f ? fmax(fmax((double)top_p, 0.0) * (double)carry, 1.0) : 0.0;
  const unsigned long long enough = sn_least(r, min_p);
  for (int i = threadIdx.x; i < n; i += SN_THREADS) {
    if (top_p < 1.f && (double)s.mass[i] >= want && (i == 0 || !((double)s.mass[i - 1] >= want))) s.ends[0] = key_at(i);
    if (min_p > 0.f) {
      const bool here = i == 0 || sn_weight_once(r, sn_value(key_at(i))) >= enough;
      const bool next = i + 1 < n && sn_weight_once(r, sn_value(key_at(i + 1))) >= enough;
      if (here && !next) s.ends[1] = key_at(i);
    }
  }
  __syncthreads();
  const unsigned last = max(kth, max(s.ends[0], s.ends[1]));
  int stay = 0;
  for (int i0 = 0; i0 < n; i0 += SN_THREADS) stay += __syncthreads_count(i0 + (int)threadIdx.x < n && key_at(i0 + threadIdx.x) >= last);
  // the first of them, by index, whose sum of weights up to it reaches the draw's share
  const unsigned long long total = s.mass[stay - 1];
  const double target = (double)total * (double)draw;
  for (int i = threadIdx.x; i < stay; i += SN_THREADS) {
    const unsigned low = (unsigned)s.list[i];    // (larger: an index before)
    unsigned long long sum = 0;
    for (int j = 0; j < stay; j++) sum += (unsigned)s.list[j] >= low ? s.mass[j] - (j ? s.mass[j - 1] : 0) : 0;
    const unsigned long long own = s.mass[i] - (i ? s.mass[i - 1] : 0);
    if (own && (double)sum >= target) atomicMin(&s.key, 0xffffffffu - low);
  }
  __syncthreads();
  return s.key == 0xffffffffu ? likeliest : (int)s.key;
}

__global__ void __launch_bounds__(SN_THREADS, 1) sample_nucleus_kernel(const SnArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  SnShared& s = *reinterpret_cast<SnShared*>(smem);
  float* kept = reinterpret_cast<float*>(smem + (sizeof(SnShared) + 15) / 16 * 16);
  pdl_launch_dependents();
  pdl_wait();
  if (a.shares > 1) cg::this_cluster().barrier_arrive();          // (nobody's shared memory is written before its CTA runs)
  const int row = blockIdx.x / a.shares, rank = blockIdx.x % a.shares, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float top_p = a.top_p[row], min_p = a.min_p[row], temperature = a.temperature[row];
  if (a.only && top_p >= 1.f && min_p <= 0.f) {                   // (the whole cluster)
    if (a.shares > 1) cg::this_cluster().barrier_wait();
    return;
  }
  const int part = ((a.V + a.shares - 1) / a.shares + 3) & ~3, first = min(rank * part, a.V);
  SnRow r;
  r.n = min(part, a.V - first);
  r.z = a.logits + row * a.ld + first;
  r.vec = a.vec;
  const int per_warp = ((r.n + SN_WARPS - 1) / SN_WARPS + 127) / 128 * 128;
  r.warp_from = min(warp * per_warp, r.n);
  r.warp_to = min(r.warp_from + per_warp, r.n);
  r.weight = nullptr;
  r.powers = s.powers;
  r.bits = a.bits;
  if (threadIdx.x == 0) s.listed = 0;
#pragma unroll
  for (int i = threadIdx.x; i < SN_POWERS / 2; i += SN_THREADS) reinterpret_cast<ulonglong2*>(s.powers)[i] = reinterpret_cast<const ulonglong2*>(sn_powers.of)[i];
  int turn = 0;

  // ---- the maximum, of equal ones the first
  float top = -INFINITY;
  int top_at = -1;                               // (none but minus infinity and no numbers)
  for (int i0 = r.warp_from + 4 * lane; i0 < r.warp_to; i0 += 128 * SN_AHEAD) {
    float v[SN_AHEAD][4];
#pragma unroll
    for (int u = 0; u < SN_AHEAD; u++) {
      v[u][0] = v[u][1] = v[u][2] = v[u][3] = -INFINITY;
      if (i0 + 128 * u < r.warp_to) sn_four(r, i0 + 128 * u, v[u]);
    }
#pragma unroll
    for (int u = 0; u < SN_AHEAD; u++) {
      const int i = i0 + 128 * u;
      if (a.keep && i < r.warp_to) *reinterpret_cast<float4*>(kept + i) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (v[u][j] > top) { top = v[u][j]; top_at = i + j; }
    }
  }
  // key above the complement of the index
  unsigned long long best = top_at < 0 ? 0ull : (unsigned long long)sn_order(top) << 32 | (0xffffffffu - (unsigned)(first + top_at));
  if (a.keep) { r.z = kept; r.vec = 1; }
  auto larger = [](unsigned long long x, unsigned long long y) { return x > y ? x : y; };
  const unsigned own = (unsigned)(best >> 32);
  best = sn_block(s, best, larger);
  if (a.shares > 1) cg::this_cluster().barrier_wait();
  const unsigned long long* words = sn_exchange(s, a.shares, best, turn);
  for (int c = 0; c < a.shares; c++) best = larger(best, words[c]);
  const int likeliest = (int)(0xffffffffu - (unsigned)best);
  r.top = sn_value((unsigned)(best >> 32));
  // (also where the row has no finite maximum: what is infinite or alone has all of the probability)
  if (!(temperature > 0.f) || !(fabsf(r.top) < INFINITY) || (unsigned)(best >> 32) == 0) {
    if (rank == 0 && threadIdx.x == 0) a.out[row] = (unsigned)(best >> 32) ? likeliest : 0;
    return;
  }
  // (a temperature of 2^-120 and below is this one: all but the largest are out of sight)
  const double c = 1.0 / (fmax((double)temperature, 7.5e-37) * 0.69314718055994530942);
  r.c = (float)c;
  r.c2 = (float)(c - (double)r.c);

  // ---- which logits stay
  unsigned floor = SN_LOWEST;
  const int k = a.top_k[row];
  if (k > 0 && k <= SN_FEW && k < a.V) {
    const int token = sn_by_list(s, r, a.shares, rank, first, k, own, top_p, min_p, a.draws[row], likeliest, turn);
    if (token >= 0) {
      if (rank == 0 && threadIdx.x == 0) a.out[row] = token;
      return;
    }
  }
  if (k > 0 && k < a.V) floor = sn_border<false>(s, r, a.shares, floor, (double)k);
  unsigned last = floor;
  if (top_p < 1.f) {
    if (a.weights) r.weight = reinterpret_cast<unsigned long long*>(kept + part);
    last = max(last, sn_border<true>(s, r, a.shares, floor, fmax((double)top_p, 0.0)));
  }
  if (min_p > 0.f) {
    const unsigned long long enough = sn_least(r, min_p);
    __syncthreads();
    if (warp == 0) {
      const unsigned top = sn_order(r.top);
      const unsigned key = sn_first_key(SN_LOWEST - 1, top, [&](unsigned k) { return k >= top || sn_weight_once(r, sn_value(k)) >= enough; });
      if (lane == 0) s.key = key;
    }
    __syncthreads();
    last = max(last, s.key);
  }

  // ---- the first of them whose running sum reaches the draw's share
  const float last_z = sn_value(last);
  auto weights = [&](int i, unsigned long long (&w)[4]) {
    float v[4];
    sn_four(r, i, v);
    w[0] = w[1] = w[2] = w[3] = 0;
    if (fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= last_z) sn_weights_at(r, i, v, last_z, w);
    return w[0] + w[1] + w[2] + w[3];
  };
  unsigned long long sum = 0, w[4];
#pragma unroll 1
  for (int i = r.warp_from + 4 * lane; i < r.warp_to; i += 128) sum += weights(i, w);
  sum = sn_block(s, sum, [](unsigned long long x, unsigned long long y) { return x + y; });
  words = sn_exchange(s, a.shares, sum, turn);
  unsigned long long total = 0, before = 0;
  for (int c = 0; c < a.shares; c++) total += words[c];
  const double target = (double)total * (double)a.draws[row];
  int owner = -1;
  for (int c = 0; c < a.shares && owner < 0; c++) {
    if (words[c] && (double)(before + words[c]) >= target) owner = c;
    else before += words[c];
  }
  if (owner < 0 && rank == 0 && threadIdx.x == 0) a.out[row] = likeliest;      // (a draw beyond its range)
  if (owner != rank) return;
  int at = 0;
  for (; at < SN_WARPS - 1 && !(s.warps[at] && (double)(before + s.warps[at]) >= target); at++) before += s.warps[at];
  if (warp != at) return;
  for (int i = r.warp_from + 4 * lane; i - 4 * lane < r.warp_to; i += 128) {
    const unsigned long long own = i < r.warp_to ? weights(i, w) : 0;
    unsigned long long incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, own && (double)(before + incl) >= target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        unsigned long long run = before + incl - own;
        int j = 0;
        while (j < 3 && !(w[j] && (double)(run + w[j]) >= target)) run += w[j++];
        a.out[row] = first + i + j;
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
}

// How many clusters of ``n`` CTAs run at a time on device ``dev``, the current one
static int sn_clusters(int n, size_t smem, int sms, int dev) {
  static int known[64][SN_MAX_SHARES + 1];
  if (known[dev][n]) return known[dev][n];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n * 1024);
  cfg.blockDim = dim3(SN_THREADS);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = n;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int got = 0;
  if (cudaOccupancyMaxActiveClusters(&got, sample_nucleus_kernel, &cfg) != cudaSuccess || got < 1) {
    (void)cudaGetLastError();
    got = sms / (2 * n);
  }
  return known[dev][n] = got;
}

// logits float32 [R, V], rows ``ld`` apart; temperature, top_p, min_p, draws float32 and top_k int32 [R]; out int32 [R].  ``only``: rows with
// neither top_p below 1 nor min_p above 0 are left as they are.
extern "C" int qd_sample_nucleus(const float* logits, long long ld, int R, int V, const float* temperature, const int* top_k, const float* top_p,
                                 const float* min_p, const float* draws, int* out, int only, int sms, cudaStream_t stream) {
  if (R <= 0) return 0;
  if (V <= 0 || V > QD_NUCLEUS_MAX_VOCABULARY || sms < 1) return QD_ERR_UNSUPPORTED;
  SnArgs a = {logits, ld, temperature, top_p, min_p, draws, top_k, out, V, 1, 0, 0, 0, V > 1 << 18 ? 40 : 44, only};
  a.vec = !((uintptr_t)logits & 15) && ld % 4 == 0;
  const size_t fixed = (sizeof(SnShared) + 15) / 16 * 16, most = fixed + SN_KEEP * 4;
  static bool allowed[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return QD_ERR_UNSUPPORTED;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(sample_nucleus_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaFuncSetAttribute(sample_nucleus_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess)
      return (int)cudaGetLastError();
    allowed[dev] = true;
  }
  // as many CTAs to a row as run at a time, with two tiles of 2,048 to each
  for (int n = 2; n <= SN_MAX_SHARES && V / n >= 4096 && R <= sn_clusters(n, most, sms, dev); n *= 2) a.shares = n;
  const int part = ((V + a.shares - 1) / a.shares + 3) & ~3;
  a.keep = part <= SN_KEEP;
  a.weights = part <= SN_KEEP / 3;                  // (8 bytes each beside 4)
  if ((long long)R * a.shares > 0x7fffffffll) return QD_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(R * a.shares));
  cfg.blockDim = dim3(SN_THREADS);
  cfg.dynamicSmemBytes = fixed + (a.keep ? (size_t)part * (a.weights ? 12 : 4) : 0);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.shares;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = qd_pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&cfg, sample_nucleus_kernel, a);
  return qd_last_error();
}
