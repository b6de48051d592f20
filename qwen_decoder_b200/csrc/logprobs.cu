// Of each row of logits z [V]: the log probability of a given token, the distribution's entropy and the most probable tokens with theirs,
// in one pass over the row:
//
//   log p_i = z_i - m - log S,   S = sum_j e^(z_j - m),   m = max_j z_j
//   H = -sum_j p_j log p_j = log S - D / S,   D = sum_j (z_j - m) e^(z_j - m)      (kept over log 2)
//
// Every thread keeps m, S and D of what it has seen (with a larger maximum, by d < 0 of the old one: S e^d and (D + d S) e^d); they are
// joined at the end.  A row is bound by its reading; few rows are shared by clusters of up to 16 CTAs, which join over their shared
// memories, so that a call is one launch without scratch memory of its own.
//
// The most probable ``top``: a token is a 64-bit key, its logit's bits in their order above the complement of its index, so that of equal
// logits the lowest index is the largest key.  While a row is read only the maximum of every 512 neighbouring logits (a warp's of a tile) is
// kept.  Then the ``top`` largest maxima are found, of equal ones the first: no other 512 hold one of the ``top`` logits, for each of those
// chosen has one that comes before all of theirs.  They are read again (20 of 2 KB of a row of 600), and what reaches the least of the chosen
// maxima is put in order by counting for each key how many are larger.  Where more than LP_HITS of 512 do (a thousand equal logits, a mask that
// leaves fewer than ``top``), their largest ``top`` are taken one by one.  (With lists that grew while the row was read, 509 rows of 152,064
// took 80 us with one to a CTA and a barrier to every tile, 131 with one to a warp; so they take 56, and 48 without any.)
// Of sorted lists of several CTAs the keys that count are those not below the least of the L lists' ceil(top / L)-th keys, which ``top`` keys
// reach.
//
// The reference has no log probabilities; its sampler's softmax is common.cpp:576-629.
#include "common.cuh"

#define LP_THREADS 256
#define LP_WARPS (LP_THREADS / 32)
#define LP_EACH 16                           // logits of a thread's tile
#define LP_TILE (LP_THREADS * LP_EACH)
#define LP_MAX_TOP QD_LOGPROBS_MAX_TOP
#define LP_MAX_SHARES 16
#define LP_CHUNK 512                         // a warp's logits of a tile
#define LP_HITS 64                           // logits of a chunk that join without being chosen one by one
#define LP_LANE 16                           // chunks to a lane of the warp that chooses
#define LP_MAX_CHUNKS (32 * LP_LANE)         // of a CTA
#define LP_MAX_VOCABULARY (LP_MAX_SHARES * (LP_MAX_CHUNKS / LP_WARPS) * LP_TILE)
static_assert(LP_MAX_VOCABULARY == QD_LOGPROBS_MAX_VOCABULARY, "what the host's side refuses");
#define LP_LOWEST (-3.402823466e38f)

struct LpArgs {
  const void* logits;
  const int* tokens;
  float *logprob, *entropy, *top_logprobs;
  int* top_ids;
  int R, V, top, shares, vec;
  long long ld;
};
struct LpSum { float m, s, d; };

__device__ __forceinline__ unsigned lp_order(float z) {
  const unsigned u = __float_as_uint(z + 0.0f);                    // (both zeros alike)
  return z != z ? 0u : u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float lp_value(unsigned order) { return __uint_as_float(order ^ (order >> 31 ? 0x80000000u : 0xffffffffu)); }
// no number has the key 0, as what lies behind the row's end
__device__ __forceinline__ unsigned long long lp_key(float z, int i) {
  const unsigned o = lp_order(z);
  return o ? (unsigned long long)o << 32 | (0xffffffffu - (unsigned)i) : 0ull;
}
// (z - m) / log 2, not below -256: 2^-256 is 0 in float32, and an infinite distance would make 0 times infinity
#define LP_LOG2E 1.4426950408889634f
#define LP_LN2 0.6931471805599453f
__device__ __forceinline__ float lp_exp2(float a) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(a));
  return e;
}
__device__ __forceinline__ void lp_to(LpSum& a, float m) {           // the sums as of a larger maximum
  const float d = fmaxf((a.m - m) * LP_LOG2E, -256.f), e = lp_exp2(d);
  a.d = (a.d + d * a.s) * e;
  a.s *= e;
  a.m = m;
}
__device__ __forceinline__ void lp_join(LpSum& a, LpSum b) {
  const float m = fmaxf(a.m, b.m);
  lp_to(a, m);
  lp_to(b, m);
  a.s += b.s;
  a.d += b.d;
}
__device__ __forceinline__ unsigned long long lp_warp_max(unsigned long long k) {
  const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(k >> 32));
  const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(k >> 32) == hi ? (unsigned)k : 0u);
  return (unsigned long long)hi << 32 | lo;
}

struct LpShared {
  unsigned long long joined[LP_MAX_TOP * LP_HITS], sorted[LP_MAX_TOP], nth[LP_MAX_SHARES];
  unsigned peaks[LP_MAX_CHUNKS], least;
  LpSum sum[LP_WARPS], whole;
  int chosen[LP_MAX_TOP], n_chosen, n_joined;
};

// Which logit a lane's i-th of 512 from ``at`` on is: whole 16 bytes of a lane side by side, or one by one
template <typename TX>
__device__ __forceinline__ int lp_index(int at, int i, bool vec) {
  constexpr int E = 16 / (int)sizeof(TX);
  const int lane = threadIdx.x & 31;
  return vec ? at + (i / E) * 32 * E + lane * E + i % E : at + i * 32 + lane;
}
// A lane's 16 of them, minus infinity behind the row's end
template <typename TX>
__device__ __forceinline__ void lp_load(float (&v)[LP_EACH], const TX* z, int at, int V, bool vec) {
  constexpr int E = 16 / (int)sizeof(TX);
  if (vec && at + LP_CHUNK <= V) {
#pragma unroll
    for (int i = 0; i < LP_EACH / E; i++) {
      const uint4 raw = *reinterpret_cast<const uint4*>(z + lp_index<TX>(at, i * E, true));
      const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int j = 0; j < E; j++)
        v[i * E + j] = __uint_as_float(sizeof(TX) == 4 ? w[j & 3] : j & 1 ? w[j >> 1 & 3] & 0xffff0000u : w[j >> 1 & 3] << 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < LP_EACH; i++) {
      const int k = lp_index<TX>(at, i, vec);
      v[i] = k < V ? to_float(z[k]) : -INFINITY;
    }
  }
}

// A warp finds the ``top`` largest of up to 32 N chunks' maxima, of equal ones the first: bit by bit the largest bound that ``top`` of
// them reach
template <int N>
__device__ __forceinline__ void lp_choose(LpShared& sh, int chunks, int top) {
  const int lane = threadIdx.x & 31;
  unsigned peak[N], high = 0, low = 0xffffffffu;                     // the largest and the least (0: no number)
#pragma unroll
  for (int i = 0; i < N; i++) {
    peak[i] = 32 * i + lane < chunks ? sh.peaks[32 * i + lane] : 0u;
    high = max(high, peak[i]);
    low = min(low, peak[i] - 1u);
  }
  high = __reduce_max_sync(0xffffffffu, high);
  low = __reduce_min_sync(0xffffffffu, low) + 1u;
  const auto reach = [&](unsigned bound) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; i++) n += peak[i] >= bound;
    return __reduce_add_sync(0xffffffffu, n);
  };
  unsigned bound = high ? low : 1u;
  int all = reach(bound), bit = 31 - __clz(high ^ low);
  if (all > top) bound = bit < 0 ? high : high & ~0u << bit << 1;    // (what they begin with alike)
#pragma unroll 1
  for (; bit >= 0 && all > top; bit--) {
    const unsigned higher = bound | 1u << bit;
    const int n = reach(higher);
    if (n >= top) {
      bound = higher;
      all = n;
    }
  }
  // (more of them than ``top`` only where some are equal to the bound)
  int taken = 0, above = 0;
  if (all > top) above = reach(bound + 1u);
  unsigned least = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const bool over = peak[i] > bound, equal = peak[i] == bound;
    unsigned take = __ballot_sync(0xffffffffu, over || equal);
    if (all > top) {
      const unsigned equals = __ballot_sync(0xffffffffu, equal);
      const int before = __popc(equals & ((1u << lane) - 1u));
      take = __ballot_sync(0xffffffffu, over || (equal && above + before < top));
      above += __popc(equals);
    }
    if (take >> lane & 1) {
      sh.chosen[taken + __popc(take & ((1u << lane) - 1u))] = 32 * i + lane;
      least = min(least, peak[i]);
    }
    taken += __popc(take);
  }
  least = __reduce_min_sync(0xffffffffu, least);
  if (lane == 0) {
    sh.n_chosen = taken;
    sh.least = taken == top ? least : 1u;
  }
}

template <typename TX>
__global__ void __launch_bounds__(LP_THREADS, 4) logprobs_kernel(const LpArgs a) {
  __shared__ LpShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x / a.shares, share = blockIdx.x - row * a.shares;
  if (threadIdx.x == 0) sh.n_joined = 0;
  pdl_launch_dependents();
  pdl_wait();
  const TX* z = (const TX*)a.logits + row * a.ld;
  const int tiles = (a.V + LP_TILE - 1) / LP_TILE;
  const int lo = (int)((long long)tiles * share / a.shares), hi = (int)((long long)tiles * (share + 1) / a.shares);
  LpSum sum = {LP_LOWEST, 0.f, 0.f};
  // (one thread asks for the token, and behind the first tile for its logit: at the end both would be waited for, 2 us)
  const bool writes = share == 0 && threadIdx.x == 0;
  int token = -1;
  float its = __uint_as_float(0x7fc00000u);
  if (writes) token = a.tokens[row];
  float next[LP_EACH];
  lp_load(next, z, lo * LP_TILE + warp * LP_CHUNK, a.V, a.vec);
  for (int tile = lo; tile < hi; tile++) {
    float v[LP_EACH];
#pragma unroll
    for (int i = 0; i < LP_EACH; i++) v[i] = next[i];
    if (tile + 1 < hi) lp_load(next, z, (tile + 1) * LP_TILE + warp * LP_CHUNK, a.V, a.vec);
    float m = v[0];
#pragma unroll
    for (int i = 1; i < LP_EACH; i++) m = fmaxf(m, v[i]);
    if (m > sum.m) lp_to(sum, m);
#pragma unroll
    for (int i = 0; i < LP_EACH; i++) {
      const float d = (v[i] - sum.m) * LP_LOG2E, e = lp_exp2(d);
      sum.s += e;                                                    // (NaN comes this way)
      sum.d = fmaf(fmaxf(d, -256.f), e, sum.d);
    }
    if (a.top) {
      const unsigned peak = __reduce_max_sync(0xffffffffu, lp_order(m));
      if (lane == 0) sh.peaks[(tile - lo) * LP_WARPS + warp] = peak;
    }
    if (writes && tile == lo && token >= 0 && token < a.V) its = to_float(z[token]);
  }
  // ---- the CTA's sums and its list
  const float m = lp_value(__reduce_max_sync(0xffffffffu, lp_order(sum.m)));
  lp_to(sum, m);
  sum.s = warp_sum(sum.s);
  sum.d = warp_sum(sum.d);
  if (lane == 0) sh.sum[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    LpSum w = sh.sum[0];
    for (int i = 1; i < LP_WARPS; i++) lp_join(w, sh.sum[i]);
    sh.whole = w;
  }
  // the joined keys in order
  auto order = [&]() {
    __syncthreads();
    const int total = sh.n_joined;
    for (int i = threadIdx.x; i < total; i += LP_THREADS) {
      const unsigned long long mine = sh.joined[i];
      int before = 0;
      for (int j = 0; j < total; j++) before += sh.joined[j] > mine;
      if (before < a.top) sh.sorted[before] = mine;
    }
    if ((int)threadIdx.x >= total && (int)threadIdx.x < a.top) sh.sorted[threadIdx.x] = 0;
    __syncthreads();
  };
  if (a.top) {
    if (warp == 0) {
      if ((hi - lo) * LP_WARPS <= 128) lp_choose<4>(sh, (hi - lo) * LP_WARPS, a.top);
      else lp_choose<LP_LANE>(sh, (hi - lo) * LP_WARPS, a.top);
    }
    __syncthreads();
    if (sh.n_chosen < a.top) {
      // Fewer chunks than tokens: of each chunk the maxima of 64 times 8 logits, of which the ``top``-th is reached by ``top`` logits
      for (int c = warp; c < sh.n_chosen; c += LP_WARPS) {
        float v[LP_EACH];
        lp_load(v, z, lo * LP_TILE + sh.chosen[c] * LP_CHUNK, a.V, a.vec);
        float x = v[0], y = v[LP_EACH / 2];
#pragma unroll
        for (int i = 1; i < LP_EACH / 2; i++) {
          x = fmaxf(x, v[i]);
          y = fmaxf(y, v[LP_EACH / 2 + i]);
        }
        unsigned one = lp_order(x), two = lp_order(y), o = 0;
        for (int k = 0; k < a.top; k++) {
          o = __reduce_max_sync(0xffffffffu, max(one, two));
          if ((int)__ffs(__ballot_sync(0xffffffffu, max(one, two) == o)) - 1 == lane) {
            if (one == o) one = 0;
            else two = 0;
          }
        }
        if (lane == 0 && o) atomicMax(&sh.least, o);
      }
      __syncthreads();
    }
    const float least = sh.least > lp_order(-INFINITY) ? lp_value(sh.least) : -INFINITY;
    const int n_chosen = sh.n_chosen;
    if (warp < n_chosen) lp_load(next, z, lo * LP_TILE + sh.chosen[warp] * LP_CHUNK, a.V, a.vec);
    for (int c = warp; c < n_chosen; c += LP_WARPS) {
      const int at = lo * LP_TILE + sh.chosen[c] * LP_CHUNK;
      float v[LP_EACH];
#pragma unroll
      for (int i = 0; i < LP_EACH; i++) v[i] = next[i];
      if (c + LP_WARPS < n_chosen) lp_load(next, z, lo * LP_TILE + sh.chosen[c + LP_WARPS] * LP_CHUNK, a.V, a.vec);
      unsigned hits = 0;
#pragma unroll
      for (int i = 0; i < LP_EACH; i++)
        if (v[i] >= least && lp_index<TX>(at, i, a.vec) < a.V) hits |= 1u << i;
      if (__reduce_add_sync(0xffffffffu, __popc(hits)) <= LP_HITS) {
        while (hits) {
          const int i = __ffs(hits) - 1;
          hits &= hits - 1;
          float x = v[0];
#pragma unroll
          for (int j = 1; j < LP_EACH; j++)
            if (j == i) x = v[j];
          sh.joined[atomicAdd(&sh.n_joined, 1)] = lp_key(x, lp_index<TX>(at, i, a.vec));
        }
      } else {
        // their largest ones, one after the other
        unsigned long long last = ~0ull;
        for (int k = 0; k < a.top; k++) {
          unsigned long long mine = 0;
#pragma unroll
          for (int i = 0; i < LP_EACH; i++) {
            const unsigned long long key = hits >> i & 1 ? lp_key(v[i], lp_index<TX>(at, i, a.vec)) : 0ull;
            if (key < last && key > mine) mine = key;
          }
          last = lp_warp_max(mine);
          if (!last) break;
          if (lane == 0) sh.joined[atomicAdd(&sh.n_joined, 1)] = last;
        }
      }
    }
    order();
  } else {
    __syncthreads();
  }
  // ---- the row's
  LpSum whole = sh.whole;
  if (a.shares > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (share == 0) {
      const unsigned base = (unsigned)__cvta_generic_to_shared(&sh);
      auto at = [&](const void* p, int cta) {
        unsigned r;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(base + (unsigned)((const char*)p - (const char*)&sh)), "r"(cta));
        return r;
      };
      // (a lane to a share, and of the lists warp w those of shares w and w + 8: all that is far is on its way together)
      unsigned long long key[LP_MAX_SHARES / LP_WARPS];
#pragma unroll
      for (int i = 0; i < LP_MAX_SHARES / LP_WARPS; i++) {
        const int c = warp + i * LP_WARPS;
        key[i] = 0;
        if (c < a.shares && lane < a.top) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key[i]) : "r"(at(&sh.sorted[lane], c)) : "memory");
      }
      if (warp == 0) {
        sum = {LP_LOWEST, 0.f, 0.f};
        if (lane < a.shares) {
          LpSum x;
          const unsigned from = at(&sh.whole, lane);
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x.m) : "r"(from) : "memory");
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x.s) : "r"(from + 4) : "memory");
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x.d) : "r"(from + 8) : "memory");
          sum = x;
        }
        lp_to(sum, lp_value(__reduce_max_sync(0xffffffffu, lp_order(sum.m))));
        whole.m = sum.m;
        whole.s = warp_sum(sum.s);
        whole.d = warp_sum(sum.d);
      }
      if (a.top) {
        const int nth = (a.top + a.shares - 1) / a.shares - 1;
#pragma unroll
        for (int i = 0; i < LP_MAX_SHARES / LP_WARPS; i++) {
          const int c = warp + i * LP_WARPS;
          const unsigned long long of = __shfl_sync(0xffffffffu, key[i], nth);
          if (lane == 0) sh.nth[c] = c < a.shares ? of : ~0ull;
        }
        if (threadIdx.x == 0) sh.n_joined = 0;
        __syncthreads();
        const unsigned long long bound = ~lp_warp_max(lane < LP_MAX_SHARES ? ~sh.nth[lane] : 0ull);
#pragma unroll
        for (int i = 0; i < LP_MAX_SHARES / LP_WARPS; i++)
          if (key[i] && key[i] >= bound) sh.joined[atomicAdd(&sh.n_joined, 1)] = key[i];
        order();
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (share) return;
  }
  if (warp) return;
  const float log_s = logf(whole.s);
  // (a row of minus infinities alone has no probabilities: none is above 0)
  auto log_p = [&](float x) { return whole.s == 0.f ? -INFINITY : x - whole.m - log_s; };
  if (threadIdx.x == 0) {
    a.logprob[row] = token >= 0 && token < a.V ? log_p(its) : its;
    a.entropy[row] = whole.s == 0.f ? 0.f : log_s - LP_LN2 * (whole.d / whole.s);
  }
  if ((int)threadIdx.x < a.top) {
    const unsigned long long key = sh.sorted[threadIdx.x];
    const bool there = key != 0;
    a.top_ids[(size_t)row * a.top + threadIdx.x] = there ? (int)(0xffffffffu - (unsigned)key) : -1;
    a.top_logprobs[(size_t)row * a.top + threadIdx.x] = there ? log_p(lp_value((unsigned)(key >> 32))) : __uint_as_float(0x7fc00000u);
  }
}

// How many clusters of ``n`` CTAs run at a time on device ``dev``, the current one
static int lp_clusters(int n, int sms, int dev) {
  static int known[64][LP_MAX_SHARES + 1];
  if (known[dev][n]) return known[dev][n];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n * 1024);
  cfg.blockDim = dim3(LP_THREADS);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = n;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int got = 0;
  if (cudaOccupancyMaxActiveClusters(&got, logprobs_kernel<float>, &cfg) != cudaSuccess || got < 1) {
    (void)cudaGetLastError();
    got = 3 * sms / n;
  }
  return known[dev][n] = got;
}

// logits [R, V] float32 or bfloat16, rows ``ld`` elements apart; tokens int32 [R] (outside of [0, V): the log probability NaN); logprob and
// entropy float32 [R]; top_ids int32 and top_logprobs float32 [R, top], top up to 32, of rows with fewer numbers -1 and NaN.
extern "C" int qd_token_logprobs(const void* logits, int dtype, long long ld, const int* tokens, float* logprob, float* entropy,
                                 int* top_ids, float* top_logprobs, int R, int V, int top, int sms, cudaStream_t stream) {
  if (R <= 0) return 0;
  if ((dtype != QD_F32 && dtype != QD_BF16) || V <= 0 || V > LP_MAX_VOCABULARY || top < 0 || top > LP_MAX_TOP || top > V || sms < 1)
    return QD_ERR_UNSUPPORTED;
  LpArgs a;
  a.logits = logits; a.tokens = tokens; a.logprob = logprob; a.entropy = entropy; a.top_ids = top_ids; a.top_logprobs = top_logprobs;
  a.R = R; a.V = V; a.top = top; a.ld = ld;
  const int size = dtype == QD_F32 ? 4 : 2;
  a.vec = !((uintptr_t)logits & 15) && ld * size % 16 == 0;
  // clusters of more than 8 are asked for once
  static bool allowed[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return QD_ERR_UNSUPPORTED;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(logprobs_kernel<float>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaFuncSetAttribute(logprobs_kernel<bf16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return (int)cudaGetLastError();
    allowed[dev] = true;
  }
  // As many CTAs to a row as run at a time, with four tiles and half again as many chunks as ``top`` to each, or two tiles where they leave a third
  // of the places free.  Measured, us, top 5: 64 rows of 152,064 with 4 and 8 16.8 and 13.4, 148 rows with 2 and 4 (some of whose clusters
  // wait) 24.7 and 30.9; 8 rows of 32,000 with 2 and 4 7.2 and 6.4, 110 rows 9.5 and 11.1; 8 rows of 151,936 with 8 and 16 7.9 and 8.6 in L2,
  // as the product over the vocabulary leaves them, 9.1 and 9.2 from memory.
  const int tiles = (V + LP_TILE - 1) / LP_TILE;
  a.shares = 1;
  for (int n = 2; n <= LP_MAX_SHARES && tiles / n >= 2 && 2 * (tiles / n) * LP_WARPS >= 3 * top; n *= 2) {
    if (tiles / n >= 4 ? R > lp_clusters(n, sms, dev) : n > 8 || 2ll * R * n > 5ll * sms) break;
    a.shares = n;
  }
  while (a.shares * (LP_MAX_CHUNKS / LP_WARPS) * LP_TILE < V) a.shares++;      // a CTA keeps so many maxima
  if ((long long)R * a.shares > 0x7fffffffll) return QD_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(R * a.shares));
  cfg.blockDim = dim3(LP_THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.shares;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = qd_pdl_enabled() ? 2 : 1;
  if (dtype == QD_F32) cudaLaunchKernelEx(&cfg, logprobs_kernel<float>, a);
  else cudaLaunchKernelEx(&cfg, logprobs_kernel<bf16>, a);
  return qd_last_error();
}
