// A token of each row of logits by temperature, top-k, top-p and min-p, from a given number r in [0, 1):
//
//   w_i = e^((z_i - max z) / T),   K = {z_i >= the k-th largest},   N = {z_i >= t}: t the largest logit with
//   sum_{K, z_i >= t} w_i >= top_p sum_K w_i,   M = {w_i >= min_p};   the first i of K, N and M whose running sum of w reaches r times all of it
//
// (logits that are equal are in or out together).  Temperature 0 is the largest logit, of equal ones the first.  The reference has
// temperature and top-k (common.cpp:576-629).
//
// Which token a number falls to, and which logit is the last of a nucleus, changes where sums are next to a border, and rows have a hundred
// thousand borders.  So weights are whole numbers, w 2^45 to within six (2^41 for rows of more than 2^18 logits): their sums are exact, in whatever
// order, and a row's token does not depend on how its work is shared.  What is lost is 3 2^-44 of the largest weight for each at most.
//
// A cluster of S CTAs shares a row, contiguous parts of it (in shared memory where they fit).  The k-th largest logit and t are found
// alike, by histograms (counts, or counts and weights) over the cluster: first over 1,409 equal steps of z below the maximum, down to 44 ln 2 T,
// where weights end (the logits of a row are spread over many of these, so that few additions meet; in steps of the number's leading bits
// they would not be); then the logits of the step that the border lies in go to one CTA, which adds up for each of them what it and those above it
// have.  Where they are more than SN_LIST (a thousand equal logits), histograms over steps of the logit's bits follow, until a step is one number.
// The draw's token is looked for in the CTA that it falls to, a sixteenth of its part, a sixteenth of that, 128 logits.
//
// A top-k of up to 256 needs none of that: the k-th largest of a CTA's threads' own maxima has k logits that reach it, as the least of the
// CTAs' ceil(k / S)-th ones has; what reaches the larger of these bounds is little more than k logits, which go to one CTA's list and decide the rest
// there.  (Rows of 152,064 with top-p 0.95, by the list and by histograms: one with k = 20 13.4 and 32.1 us, with 250 32.1 and 32.4, with 500 98
// and 33; 64 with k = 20 17.5 and 92, with 250 43 and 93, with 500 122 and 94.)
//
// 64 rows of 152,064 take 20 us with k of up to 100, top-p and min-p, of which 6 are their 39 MB at the rate of device memory; then bound by trips over
// the cluster (1.5 to 3 thousand cycles each) and the list's sums.  By top-p alone 82 (122 with a top-p of 0.925 to 0.975, row by row), by min-p alone 31.  By top-p bound by the weights' arithmetic, 55 instructions for each logit,
// a third of them on whole numbers at half the rate, and their two additions in shared memory (40 us with the rows and no weights).  One row of
// 151,936 by top-p 25, S = 16: seven trips over the cluster and code that runs once, out of the reach of the instructions' caches.
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
#define SN_OCTAVES 44                            // below the maximum a weight is 0
#define SN_STEP 7                                // log2 of the powers to a step of the first histogram
#define SN_DOWN 18                               // what a power is shifted by at the maximum: 2^63 over 2^45
static_assert((SN_OCTAVES * SN_POWERS >> SN_STEP) + 1 < SN_BINS, "steps of the first histogram");
#define SN_FEW 256                               // a top-k up to here goes by the list
#define SN_LIST 1024
#define SN_AHEAD 4                               // 16 bytes each that a thread has on their way

struct SnArgs {
  const float* logits;
  long long ld;
  const float *temperature, *top_p, *min_p, *draws;
  const int* top_k;
  int* out;
  int V, shares, vec, keep, maxima, wide, only;           // in shared memory: a CTA's logits, the maxima of a thread's 16; wide: octaves that weights are smaller by
};
// 2^(-k / 4096) over 2^63: powers of the twelfth root of a half, each root the whole root of the one before, over 2^63
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
      of[k] = p;
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
    struct {                                     // logits that go to the cluster's first CTA, of a small top-k or of the step that a border lies in: keys (of a
      unsigned long long list[SN_LIST], mass[SN_LIST];       // top-k above the complement of their index); their weights
    };
  };
  __align__(16) unsigned long long powers[SN_POWERS];
  unsigned near[SN_LIST];                        // (the step's keys: they come while the histogram is still there)
  int listed;
  unsigned long long got[2][SN_MAX_SHARES];      // a word of each CTA
  unsigned long long warps[SN_WARPS], above;
  unsigned bin, ends[2], key, token, last_step[2], counts[SN_WARPS];
  float kept[SN_WARPS][160];                     // what a warp has found, up to 31 of before and 128
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
  float base, octaves;                           // what is added to z's distance in 8 SN_POWERS-ths of an octave; of them until weights end
  unsigned first_step;
  const unsigned long long* powers;              // in shared memory
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
// SN_AHEAD times four, 128 apart
__device__ __forceinline__ void sn_ahead(const SnRow& r, int i, float (&v)[SN_AHEAD][4]) {
#pragma unroll
  for (int u = 0; u < SN_AHEAD; u++) {
    v[u][0] = v[u][1] = v[u][2] = v[u][3] = -INFINITY;
    if (i + 128 * u < r.warp_to) sn_four(r, i + 128 * u, v[u]);
  }
}
// z's place: eight times the whole number j of 4,096ths next above y = (max - z) / (T log 2) (or the one behind that), as the bits of a float32 number of
// 2^23 and more that has ``base`` for 0, whose octaves are SN_DOWN and more.  0 where weights have ended, and for what is no number.
__device__ __forceinline__ unsigned sn_place(const SnRow& r, float z) {
  const float p = (r.top - z) * r.c;
  return p < r.octaves ? __float_as_uint(fmaf(p, 8.f * SN_POWERS, r.base + 8.f)) & ~7u : 0u;
}
// steps of the first histogram: 128 of them; none (SN_BINS and more) for what has no place
__device__ __forceinline__ unsigned sn_step(const SnRow& r, unsigned place) { return (place >> (SN_STEP + 3)) - r.first_step; }
// e^((z - max) / T) over 2^-45 (2^-41 for long rows) as a whole number, -5.2 to 1.2 of it off, in 32-bit arithmetic (an instruction of 64-bit
// floating point is some 20 cycles of a scheduler; whole numbers go through at half of floating point's rate).  With d = max - z and
// c = 1 / (T log 2), each a sum of two float32 numbers, y = c d is one to 2^-47 of itself; x / log 2 = j / 4096 - y is what the place lies behind it,
// up to 8.7 / 32768, and the result is 2^(-j / 4096) (1 + x + x^2 / 2 + x^3 / 6), of a power with 31 bits beside x.
__device__ __forceinline__ unsigned long long sn_weight(const SnRow& r, float z, unsigned place) {
  const float d = r.top - z, back = d - r.top, d2 = (r.top - (d - back)) - (z + back);       // (what the difference lost)
  const float p = d * r.c;
  const float e = fmaf(d2, r.c, fmaf(d, r.c2, fmaf(d, r.c, -p)));
  const float j = (__uint_as_float(place) - r.base) * (1.f / (8 * SN_POWERS)), f = j - p, y = f - e, y2 = ((f - y) - e) + ((j - f) - p);
  const float x = y * 0.693147182f, x2 = fmaf(y2, 0.693147182f, fmaf(y, -1.90465421e-9f, fmaf(y, 0.693147182f, -x)));
  const float a = fmaf(x, 2147483648.f, 12582912.f), left = fmaf(a - 12582912.f, -1.f / 2147483648.f, x);
  const float b = fmaf(left + fmaf(x * x, fmaf(x, 1.f / 6, 0.5f), x2), 17592186044416.f, 12582912.f);
  const unsigned more = (__float_as_uint(a) << 13) + __float_as_uint(b) - ((0x4b400000u << 13) + 0x4b400000u);               // e^x - 1 over 2^-44
  const unsigned long long w = *reinterpret_cast<const unsigned long long*>(reinterpret_cast<const unsigned char*>(r.powers) + (place & 8 * (SN_POWERS - 1)));
  return (w + ((w >> 32) * more >> 12)) >> (place >> 15 & 63);
}
// (one copy of the code for what is asked for seldom: a launch goes through most of its code once, and waits for it where it is long)
__device__ __noinline__ unsigned long long sn_weight_once(const SnRow& r, float z) {
  const unsigned place = sn_place(r, z);
  return place ? sn_weight(r, z, place) : 0;
}
// a share of a sum, in whole weights, ``least`` or more
__device__ __forceinline__ unsigned long long sn_part(unsigned long long total, float share, unsigned long long least) {
  return max(__double2ull_ru(fmax((double)share, 0.0) * (double)total), least);
}
// the least weight that min_p leaves
__device__ __forceinline__ unsigned long long sn_least(const SnRow& r, float min_p) {
  return sn_part(sn_weight_once(r, r.top), fminf(min_p, 1.f), 0);
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

// Threads to each of n numbers of a list, neighbours, so that the block has them all in one or two turns
__device__ __forceinline__ int sn_threads(int n) { return n <= SN_THREADS / 8 ? 8 : n <= SN_THREADS / 4 ? 4 : n <= SN_THREADS / 2 ? 2 : 1; }
// the sum of the words of those of a list's n that ``with`` holds for, by the ``each`` threads of a number (n^2 additions, n being some hundred: less
// than putting them in order, whose steps wait for one another)
template <typename W, typename F>
__device__ __forceinline__ W sn_sum_with(int n, int each, F word) {
  W sum = 0;
#pragma unroll 4
  for (int j = threadIdx.x & (each - 1); j < n; j += each) sum += word(j);
  for (int o = each / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
// a logit of the step that a border lies in, to the list
__device__ __noinline__ void sn_put(const SnRow& r, float z, unsigned bin, int* count, unsigned* near) {
  if (sn_step(r, sn_place(r, z)) != bin) return;
  const int at = atomicAdd(count, 1);
  if (at < SN_LIST) near[at] = sn_order(z);
}
// The border among the n keys of ``near``, above all of which lies ``above``.
template <bool MASS>
__device__ unsigned sn_among(SnShared& s, const SnRow& r, int n, unsigned long long above, unsigned long long want) {
  for (int i = threadIdx.x; i < n; i += SN_THREADS) s.mass[i] = MASS ? sn_weight_once(r, sn_value(s.near[i])) : 1ull;
  if (threadIdx.x == 0) s.token = 0;
  __syncthreads();
  const int each = sn_threads(n);
  for (int i0 = 0; i0 < n; i0 += SN_THREADS / each) {
    const int i = i0 + threadIdx.x / each;
    const unsigned own = s.near[min(i, n - 1)];
    const unsigned long long sum = sn_sum_with<unsigned long long>(n, each, [&](int j) { return s.near[j] >= own ? s.mass[j] : 0ull; });
    if (i < n && above + sum >= want) atomicMax(&s.token, own);
  }
  __syncthreads();
  return s.token;
}

// The largest key t so that the logits of keys from t on, none below ``floor`` among them, hold ``want`` or more: counts, or of weights
// ``share`` of them all.  ``floor`` where there is less than that down to where weights end.
template <bool MASS>
__device__ unsigned sn_border(SnShared& s, const SnRow& r, int shares, unsigned floor, float share, unsigned long long want) {
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
    float next[4];
    if (r.warp_from + 4 * lane < r.warp_to) sn_four(r, r.warp_from + 4 * lane, next);
#pragma unroll 1
    for (int i = r.warp_from + 4 * lane; i < r.warp_to; i += 128) {
      float v[4];
      unsigned bin[4];
      unsigned long long w[4] = {1, 1, 1, 1};
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = next[j];
      if (i + 128 < r.warp_to) sn_four(r, i + 128, next);
      if (level == 0) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const unsigned place = v[j] >= from_z ? sn_place(r, v[j]) : 0u;
          bin[j] = sn_step(r, place);
          if (MASS) w[j] = sn_weight(r, v[j], place);      // (of no use without a place)
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          bin[j] = v[j] >= from_z && v[j] <= to_z ? (k_hi - sn_order(v[j])) >> shift : SN_BINS;
          if (MASS && bin[j] < SN_BINS) w[j] = sn_weight_once(r, v[j]);
        }
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
    if (MASS && level == 0) want = sn_part(total, share, 1);
    if (run < want && run + sum >= want) {
      int u = 0;
      while (u < SN_EACH - 1 && run + own[u] < want) run += own[u++];
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
      unsigned* near = shares > 1 ? cg::this_cluster().map_shared_rank(s.near, 0) : s.near;
      // (about where the step lies, its ends a 64th of it further out and by what the terms of y can have lost: few are looked at closely)
      const float wide = (float)(1 << SN_STEP) / SN_POWERS / r.c, out = wide * (1.f / 64) + fabsf(r.top) * 2.4e-7f + ((float)bin + 1.f) * wide * 2.4e-7f;
      const float lo_z = fmaxf(from_z, r.top - ((float)bin + 1.f) * wide - out), hi_z = fminf(to_z, r.top - (float)bin * wide + out);
      for (int i0 = r.warp_from + 4 * lane; i0 < r.warp_to; i0 += 128 * SN_AHEAD) {
        float v[SN_AHEAD][4];
        sn_ahead(r, i0, v);
#pragma unroll
        for (int u = 0; u < SN_AHEAD; u++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (v[u][j] >= lo_z && v[u][j] <= hi_z) sn_put(r, v[u][j], bin, count, near);
      }
      if (shares > 1) cg::this_cluster().sync();
      else __syncthreads();
      const int n = *count;
      if (n <= SN_LIST && (shares == 1 || cg::this_cluster().block_rank() == 0)) {
        const unsigned key = sn_among<MASS>(s, r, n, above, want);
        if ((int)threadIdx.x < shares) *(shares > 1 ? cg::this_cluster().map_shared_rank(&s.key, threadIdx.x) : &s.key) = key;
        __syncthreads();
      }
      if (shares > 1) cg::this_cluster().sync();           // (the first CTA's list has been counted, too)
      else __syncthreads();
      if (threadIdx.x == 0) s.listed = 0;
      if (n <= SN_LIST) return s.key;
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
          const unsigned step = sn_step(r, sn_place(r, sn_value(key)));
          return key > top || (warp ? step < bin : step <= bin);
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
__device__ int sn_by_list(SnShared& s, const SnRow& r, int shares, int rank, int first, int k, unsigned best, const float* maxima, float top_p, float min_p, float draw,
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
  // (first which of a thread's sixteens have some, then those: few have, and a turn of the whole warp for each is a trip to memory)
  const int mine = r.warp_from + 4 * lane, runs = (r.warp_to - mine + 128 * SN_AHEAD - 1) / (128 * SN_AHEAD);
  for (int t0 = 0; t0 < runs; t0 += 32) {
    unsigned has = 0;
    for (int t = t0; t < min(t0 + 32, runs); t++)
      if (!maxima || maxima[t * SN_THREADS + threadIdx.x] >= bound_z) has |= 1u << (t - t0);
    for (; has; has &= has - 1) {
      const int i0 = mine + (t0 + __ffs(has) - 1) * 128 * SN_AHEAD;
      float v[SN_AHEAD][4];
      sn_ahead(r, i0, v);
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
  // weights of those with less than k larger ones
  auto key_at = [&](int i) { return (unsigned)(s.list[i] >> 32); };
  if (threadIdx.x == 0) { s.key = 0; s.token = 0xffffffffu; }
  __syncthreads();
  const int each = sn_threads(n), turns = SN_THREADS / each, part = threadIdx.x & (each - 1);
  for (int i0 = 0; i0 < n; i0 += turns) {
    const int i = i0 + threadIdx.x / each;
    const unsigned own = key_at(min(i, n - 1));
    const int larger = sn_sum_with<int>(n, each, [&](int j) { return key_at(j) > own ? 1 : 0; });
    if (i < n && part == 0) s.mass[i] = larger < k ? sn_weight_once(r, sn_value(own)) : 0ull;
  }
  __syncthreads();
  // the last key of the nucleus: the largest with enough of the weights at it and above
  if (top_p < 1.f) {
    const unsigned long long want = sn_part(sn_sum_with<unsigned long long>(n, 32, [&](int j) { return s.mass[j]; }), top_p, 1);
    for (int i0 = 0; i0 < n; i0 += turns) {
      const int i = i0 + threadIdx.x / each;
      const unsigned own = key_at(min(i, n - 1));
      const unsigned long long sum = sn_sum_with<unsigned long long>(n, each, [&](int j) { return key_at(j) >= own ? s.mass[j] : 0ull; });
      if (i < n && sum >= want) atomicMax(&s.key, own);
    }
    __syncthreads();
  }
  const unsigned long long enough = min_p > 0.f ? sn_least(r, min_p) : 0ull;
  for (int i = threadIdx.x; i < n; i += SN_THREADS)
    if (key_at(i) < s.key || s.mass[i] < enough) s.mass[i] = 0;
  __syncthreads();
  // the first of them, by index, whose sum of weights up to it reaches the draw's share
  const unsigned long long want = sn_part(sn_sum_with<unsigned long long>(n, 32, [&](int j) { return s.mass[j]; }), draw, 1);
  for (int i0 = 0; i0 < n; i0 += turns) {
    const int i = i0 + threadIdx.x / each;
    const unsigned low = (unsigned)s.list[min(i, n - 1)];            // (larger: an index before)
    const unsigned long long sum = sn_sum_with<unsigned long long>(n, each, [&](int j) { return (unsigned)s.list[j] >= low ? s.mass[j] : 0ull; });
    if (i < n && s.mass[i] && sum >= want) atomicMin(&s.token, 0xffffffffu - low);
  }
  __syncthreads();
  return s.token == 0xffffffffu ? likeliest : (int)s.token;
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
  r.powers = s.powers;
  r.base = 12582912.f + (float)(SN_DOWN + a.wide) * 8 * SN_POWERS;
  r.octaves = (float)(SN_OCTAVES - a.wide);
  r.first_step = __float_as_uint(r.base) >> (SN_STEP + 3);
  if (threadIdx.x == 0) s.listed = 0;
#pragma unroll
  for (int i = threadIdx.x; i < SN_POWERS / 2; i += SN_THREADS) reinterpret_cast<ulonglong2*>(s.powers)[i] = reinterpret_cast<const ulonglong2*>(sn_powers.of)[i];
  int turn = 0;

  // ---- the maximum, of equal ones the first
  float top = -INFINITY;
  int top_at = -1;                               // (none but minus infinity and no numbers)
  float* most = kept + threadIdx.x;
  for (int i0 = r.warp_from + 4 * lane; i0 < r.warp_to; i0 += 128 * SN_AHEAD, most += SN_THREADS) {
    float v[SN_AHEAD][4], here = -INFINITY;
    int here_at = -1;
    sn_ahead(r, i0, v);
#pragma unroll
    for (int u = 0; u < SN_AHEAD; u++) {
      const int i = i0 + 128 * u;
      if (a.keep && i < r.warp_to) *reinterpret_cast<float4*>(kept + i) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (v[u][j] > here) { here = v[u][j]; here_at = i + j; }
    }
    if (a.maxima) *most = here;
    if (here > top) { top = here; top_at = here_at; }
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
  // 1 / (T log 2) as a pair: the quotient of one of 32 bits, and what it lacks
  const float up = temperature < 8.7e-19f ? 1.15292150e18f : 1.f, t = fmaxf(temperature, 7.5e-37f) * up;               // (2^60)
  const float t1 = t * 0.693147182f, t2 = fmaf(t, 0.693147182f, -t1) + t * -1.90465421e-9f;
  const float c1 = 1.f / t1;
  r.c = c1 * up;
  r.c2 = c1 * fmaf(-c1, t2, fmaf(-c1, t1, 1.f)) * up;

  // ---- which logits stay
  unsigned floor = SN_LOWEST;
  const int k = a.top_k[row];
  if (k > 0 && k <= SN_FEW && k < a.V) {
    const int token = sn_by_list(s, r, a.shares, rank, first, k, own, a.maxima ? kept : nullptr, top_p, min_p, a.draws[row], likeliest, turn);
    if (token >= 0) {
      if (rank == 0 && threadIdx.x == 0) a.out[row] = token;
      return;
    }
  }
  if (k > 0 && k < a.V) floor = sn_border<false>(s, r, a.shares, floor, 0.f, k);
  unsigned last = floor;
  if (top_p < 1.f) last = max(last, sn_border<true>(s, r, a.shares, floor, top_p, 0));
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

  // ---- the first of them whose running sum reaches the draw's share: the CTA that it falls to, a sixteenth of its part, of that, ..., 128 logits
  const float last_z = sn_value(last);
  unsigned long long before = 0, want = 0;
  int lo = 0, hi = r.n;
  float* found = s.kept[warp];
  for (bool whole = true;; whole = false) {
    const int per = ((hi - lo + SN_WARPS - 1) / SN_WARPS + 127) / 128 * 128, from = min(lo + warp * per, hi), to = min(from + per, hi);
    // weights of what stays, 32 at a time: few do, and those lie apart
    unsigned long long sum = 0;
    int held = 0;
#pragma unroll 1
    for (int i = from; i < to || held; i += 128) {
      if (i < to) {
        float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (i + 4 * lane < to) sn_four(r, i + 4 * lane, v);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const bool stays = i + 4 * lane + j < to && v[j] >= last_z;
          const unsigned all = __ballot_sync(0xffffffffu, stays);
          if (stays) found[held + __popc(all & ((1u << lane) - 1))] = v[j];
          held += __popc(all);
        }
        __syncwarp();
      }
      while (held >= 32 || (held && i + 128 >= to)) {
        const int n = min(held, 32);
        held -= n;
        const float z = found[held + min(lane, n - 1)];
        const unsigned place = sn_place(r, z);
        if (lane < n && place) sum += sn_weight(r, z, place);
      }
      __syncwarp();
    }
    sum = sn_block(s, sum, [](unsigned long long x, unsigned long long y) { return x + y; });
    if (whole) {
      words = sn_exchange(s, a.shares, sum, turn);
      unsigned long long total = 0;
      for (int c = 0; c < a.shares; c++) total += words[c];
      want = sn_part(total, a.draws[row], 1);
      int owner = -1;
      for (int c = 0; c < a.shares && owner < 0; c++) {
        if (before + words[c] >= want) owner = c;
        else before += words[c];
      }
      if (owner < 0 && rank == 0 && threadIdx.x == 0) a.out[row] = likeliest;  // (a draw beyond its range)
      if (owner != rank) return;
    }
    int at = 0;
    for (; at < SN_WARPS - 1 && before + s.warps[at] < want; at++) before += s.warps[at];
    lo = min(lo + at * per, hi);
    hi = min(lo + per, hi);
    if (hi - lo <= 128) break;
  }
  if (warp) return;
  float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  unsigned long long w[4], own_sum = 0;
  if (lo + 4 * lane < hi) sn_four(r, lo + 4 * lane, v);
#pragma unroll 1
  for (int j = 0; j < 4; j++) {
    w[j] = lo + 4 * lane + j < hi && v[j] >= last_z ? sn_weight_once(r, v[j]) : 0;
    own_sum += w[j];
  }
  unsigned long long incl = own_sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  const unsigned hit = __ballot_sync(0xffffffffu, before + incl >= want);
  if (hit && lane == __ffs(hit) - 1) {
    unsigned long long run = before + incl - own_sum;
    int j = 0;
    while (j < 3 && run + w[j] < want) run += w[j++];
    a.out[row] = first + lo + 4 * lane + j;
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
  SnArgs a = {logits, ld, temperature, top_p, min_p, draws, top_k, out, V, 1, 0, 0, 0, V > 1 << 18 ? 4 : 0, only};
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
  // as many CTAs to a row as run at a time, with 4,096 logits or more to each (by top-p, S = 1, 2, 4, 8, 16: one row of 151,936 134, 79, 48, 30, 25 us, 16 of
  // them 138, 80, 49, where no more than 4 run at a time; one of 32,000 34, 24, 18.3, 17.2, 17.7; of 8,000 16.0, 16.1, 14.4, and with k = 50 9.1, 10.7, 11.1)
  for (int n = 2; n <= SN_MAX_SHARES && V / n >= 4096 && R <= sn_clusters(n, most, sms, dev); n *= 2) a.shares = n;
  const int part = ((V + a.shares - 1) / a.shares + 3) & ~3;
  a.keep = part <= SN_KEEP;
  const size_t per_warp = ((size_t)(part + SN_WARPS - 1) / SN_WARPS + 127) / 128 * 128, turns = (per_warp + 128 * SN_AHEAD - 1) / (128 * SN_AHEAD);
  a.maxima = !a.keep && turns * SN_THREADS <= SN_KEEP;
  if ((long long)R * a.shares > 0x7fffffffll) return QD_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(R * a.shares));
  cfg.blockDim = dim3(SN_THREADS);
  cfg.dynamicSmemBytes = fixed + (a.keep ? part : a.maxima ? turns * SN_THREADS : 0) * 4;
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
