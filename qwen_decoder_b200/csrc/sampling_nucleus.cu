// A token of each row of logits by temperature, top-k, top-p and min-p, from a given number r in [0, 1):
//
//   w_i = e^((z_i - max z) / T),   K = {z_i >= the k-th largest},   N = {z_i >= t}: t the largest logit with
//   sum_{K, z_i >= t} w_i >= top_p sum_K w_i,   M = {w_i >= min_p};   the first i of K, N and M whose running sum of w reaches r times all of it
//
// (logits that are equal are in or out together).  Temperature 0 is the largest logit, of equal ones the first.  The reference has
// temperature and top-k (common.cpp:576-629).
//
// Which token a number falls to, and which logit is the last of a nucleus, changes where sums are next to a border, and rows have a hundred
// thousand borders.  So weights are whole numbers, w 2^44 rounded from float64 (2^40 for rows of more than 2^18 logits): their sums are exact,
// in whatever order, and a row's token does not depend on how its work is shared.  What is lost is 2^-45 of the largest weight for each.
//
// A cluster of S CTAs shares a row, contiguous parts of it (in shared memory where they fit).  The k-th largest logit and t are found
// alike, by histograms (counts, or counts and weights) over the cluster: first over 2,048 equal steps of z below the maximum, down to 45 ln 2 T,
// where weights end (the logits of a row are spread over many of these, so that few additions meet; in steps of the number's leading bits
// they would not be), then over steps of the logit's bits within the step that the border lies in, until a step is one number.
// Bound by the row's reading for the rest and by the trips over the cluster, two to a histogram.
#include "common.cuh"
#include <cooperative_groups.h>
#include <math.h>

namespace cg = cooperative_groups;

#define SN_THREADS 512
#define SN_WARPS (SN_THREADS / 32)
#define SN_BINS 2048
#define SN_EACH (SN_BINS / SN_THREADS)
#define SN_MAX_SHARES 16
#define SN_KEEP 40960                            // logits that a CTA holds in shared memory
#define SN_SPAN 31.2                             // 45 ln 2, rounded up

struct SnArgs {
  const float* logits;
  long long ld;
  const float *temperature, *top_p, *min_p, *draws;
  const int* top_k;
  int* out;
  int V, shares, vec, keep, bits, only;
};
struct SnBins { unsigned lo[SN_BINS], hi[SN_BINS]; };                 // a 64-bit sum each; counts in lo
struct SnShared {
  SnBins mine;
  unsigned long long all[SN_BINS];               // of the cluster
  unsigned long long got[2][SN_MAX_SHARES];      // a word of each CTA
  unsigned long long warps[SN_WARPS], above;
  unsigned bin, ends[2], key;
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
  float top, step;                               // the maximum; steps of the first histogram per unit of z
  double per_t, unit;                            // 1 / T; 2^bits
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
__device__ __forceinline__ double sn_exp(const SnRow& r, float z) { return exp(((double)z - (double)r.top) * r.per_t); }
__device__ __forceinline__ unsigned long long sn_weight(const SnRow& r, float z) { return (unsigned long long)__double2ll_rn(sn_exp(r, z) * r.unit); }
__device__ __forceinline__ unsigned sn_step(const SnRow& r, float z) { return (unsigned)fminf((r.top - z) * r.step, (float)SN_BINS); }

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
    for (int b = threadIdx.x; b < SN_BINS; b += SN_THREADS) s.mine.lo[b] = s.mine.hi[b] = 0;
    __syncthreads();
    for (int i = r.warp_from + 4 * lane; i < r.warp_to; i += 128) {
      float v[4];
      sn_four(r, i, v);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const unsigned key = sn_order(v[j]);
        if (key < k_lo || key > k_hi) continue;
        const unsigned bin = level ? (k_hi - key) >> shift : sn_step(r, v[j]);
        if (bin >= SN_BINS) continue;
        if (MASS) {
          const unsigned long long w = sn_weight(r, v[j]);
          const unsigned lo = (unsigned)w, hi = (unsigned)(w >> 32) + (atomicAdd(&s.mine.lo[bin], lo) > 0xffffffffu - lo ? 1u : 0u);
          if (hi) atomicAdd(&s.mine.hi[bin], hi);
        } else {
          atomicAdd(&s.mine.lo[bin], 1u);
        }
      }
    }
    if (shares > 1) {
      cg::cluster_group cl = cg::this_cluster();
      cl.sync();
      const int per = SN_BINS / shares, b0 = (int)cl.block_rank() * per;
      for (int b = b0 + (int)threadIdx.x; b < b0 + per; b += SN_THREADS) {
        unsigned long long sum = 0;
        for (int c = 0; c < shares; c++) {
          const SnBins* from = cl.map_shared_rank(&s.mine, c);
          sum += ((unsigned long long)from->hi[b] << 32) + from->lo[b];
        }
        for (int c = 0; c < shares; c++) *cl.map_shared_rank(&s.all[b], c) = sum;
      }
      cl.sync();
    } else {
      __syncthreads();
      for (int b = threadIdx.x; b < SN_BINS; b += SN_THREADS) s.all[b] = ((unsigned long long)s.mine.hi[b] << 32) + s.mine.lo[b];
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

__global__ void __launch_bounds__(SN_THREADS) sample_nucleus_kernel(const SnArgs a) {
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
  int turn = 0;

  // ---- the maximum, of equal ones the first
  unsigned long long best = 0;                   // key above the complement of the index
#pragma unroll 4
  for (int i = r.warp_from + 4 * lane; i < r.warp_to; i += 128) {
    float v[4];
    sn_four(r, i, v);
    if (a.keep) *reinterpret_cast<float4*>(kept + i) = make_float4(v[0], v[1], v[2], v[3]);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const unsigned long long k = (unsigned long long)sn_order(v[j]) << 32 | (0xffffffffu - (unsigned)(first + i + j));
      if (i + j < r.n && k > best) best = k;
    }
  }
  if (a.keep) { r.z = kept; r.vec = 1; }
  auto larger = [](unsigned long long x, unsigned long long y) { return x > y ? x : y; };
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
  r.per_t = 1.0 / (double)temperature;
  r.unit = (double)(1ull << a.bits);
  r.step = (float)fmin(SN_BINS / SN_SPAN * r.per_t, 3e38);

  // ---- which logits stay
  unsigned floor = SN_LOWEST;
  const int k = a.top_k[row];
  if (k > 0 && k < a.V) floor = sn_border<false>(s, r, a.shares, floor, (double)k);
  unsigned last = floor;
  if (top_p < 1.f) last = max(last, sn_border<true>(s, r, a.shares, floor, fmax((double)top_p, 0.0)));
  if (min_p > 0.f) {
    __syncthreads();
    if (warp == 0) {
      const unsigned top = sn_order(r.top);
      const unsigned key = sn_first_key(SN_LOWEST - 1, top, [&](unsigned k) { return k >= top || sn_exp(r, sn_value(k)) >= (double)min_p; });
      if (lane == 0) s.key = key;
    }
    __syncthreads();
    last = max(last, s.key);
  }

  // ---- the first of them whose running sum reaches the draw's share
  auto weights = [&](int i, unsigned long long (&w)[4]) {
    float v[4];
    sn_four(r, i, v);
    unsigned long long sum = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      w[j] = sn_order(v[j]) >= last ? sn_weight(r, v[j]) : 0;
      sum += w[j];
    }
    return sum;
  };
  unsigned long long sum = 0, w[4];
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
  SnArgs a = {logits, ld, temperature, top_p, min_p, draws, top_k, out, V, 1, 0, 0, V > 1 << 18 ? 40 : 44, only};
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
  if ((long long)R * a.shares > 0x7fffffffll) return QD_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(R * a.shares));
  cfg.blockDim = dim3(SN_THREADS);
  cfg.dynamicSmemBytes = fixed + (a.keep ? (size_t)part * 4 : 0);
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
