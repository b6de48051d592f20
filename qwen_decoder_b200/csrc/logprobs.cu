// Of each row of logits z [V]: the log probability of a given token, the distribution's entropy and the most probable tokens with theirs,
// in one pass over the row:
//
//   log p_i = z_i - m - log S,   S = sum_j e^(z_j - m),   m = max_j z_j
//   H = -sum_j p_j log p_j = log S - D / S,   D = sum_j (z_j - m) e^(z_j - m)
//
// Every thread keeps m, S and D of what it has seen (with a larger maximum, by d < 0 of the old one: S e^d and (D + d S) e^d); they are
// joined at the end.  A row is bound by its reading; few rows are shared by clusters of up to eight CTAs, which join over their shared
// memories, so that a call is one launch without scratch memory of its own.
//
// The most probable ``top``: a token is a 64-bit key, its logit's bits in their order above the complement of its index, so that of equal
// logits the lowest index is the largest key.  A CTA keeps a list of up to LP_LIST keys in shared memory and a threshold that at least
// ``top`` logits of the list reach; only larger ones join the list (the tokens of later tiles have higher indices: equal ones lose), which
// is cut back to its first ``top`` when it has LP_CUT.  For the first tile the threshold comes from the threads' own maxima: ``r`` of each of
// 8 warps' 32 with 8 r >= top.  Where a tile brings more than the list holds (rows in rising order, a thousand equal logits), its largest
// ``top`` are taken one by one.
//
// The reference has no log probabilities; its sampler's softmax is common.cpp:576-629.
#include "common.cuh"

#define LP_THREADS 256
#define LP_WARPS (LP_THREADS / 32)
#define LP_EACH 16                           // logits of a thread's tile
#define LP_TILE (LP_THREADS * LP_EACH)
#define LP_MAX_TOP 32
#define LP_LIST 256
#define LP_CUT 128
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
// max(z - m, -256): e^-256 is 0 in float32, and an infinite distance would make 0 times infinity; NaN stays
__device__ __forceinline__ float lp_distance(float z, float m) {
  float d = z - m;
  asm("max.NaN.f32 %0, %0, 0fC3800000;" : "+f"(d));
  return d;
}
__device__ __forceinline__ void lp_to(LpSum& a, float m) {           // the sums as of a larger maximum
  const float d = lp_distance(a.m, m), e = __expf(d);
  a.d = (a.d + d * a.s) * e;
  a.s *= e;
  a.m = m;
}
__device__ __forceinline__ unsigned long long lp_warp_max(unsigned long long k) {
  const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(k >> 32));
  const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(k >> 32) == hi ? (unsigned)k : 0u);
  return (unsigned long long)hi << 32 | lo;
}

struct LpShared {
  unsigned long long list[LP_LIST], sorted[LP_MAX_TOP], best[2][LP_WARPS];
  LpSum sum[LP_WARPS], whole;
  unsigned bound[LP_WARPS];
  int joined[3], n;
};

// The list's first ``top`` in order, as its new contents; their number.  All threads; begins and ends with a barrier.
__device__ __forceinline__ int lp_cut(LpShared& sh, int n, int top) {
  if (threadIdx.x < LP_MAX_TOP) sh.sorted[threadIdx.x] = 0;
  __syncthreads();
  if ((int)threadIdx.x < n) {
    const unsigned long long mine = sh.list[threadIdx.x];
    int before = 0;
    for (int j = 0; j < n; j++) before += sh.list[j] > mine;
    if (before < top) sh.sorted[before] = mine;
  }
  __syncthreads();
  const int left = min(n, top);
  if ((int)threadIdx.x < left) sh.list[threadIdx.x] = sh.sorted[threadIdx.x];
  __syncthreads();
  return left;
}

template <typename TX>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(const LpArgs a) {
  __shared__ LpShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x / a.shares, share = blockIdx.x - row * a.shares;
  if (threadIdx.x < 3) sh.joined[threadIdx.x] = 0;
  pdl_launch_dependents();
  pdl_wait();
  const TX* z = (const TX*)a.logits + row * a.ld;
  const int tiles = (a.V + LP_TILE - 1) / LP_TILE;
  const int lo = (int)((long long)tiles * share / a.shares), hi = (int)((long long)tiles * (share + 1) / a.shares);
  constexpr int E = 16 / (int)sizeof(TX);                            // of a load
  LpSum sum = {LP_LOWEST, 0.f, 0.f};
  float least = 0.f;                                                 // a logit joins the list above this, ...
  bool any = true;                                                   // ... or any as large in the first tile
  int n = 0;                                                         // of the list
  __syncthreads();
  for (int tile = lo; tile < hi; tile++) {
    const int t0 = tile * LP_TILE;
    // which logit a thread's i-th is: whole 16 bytes of a thread side by side, or one by one
    auto index = [&](int i) { return a.vec ? t0 + (i / E) * LP_THREADS * E + (int)threadIdx.x * E + i % E : t0 + i * LP_THREADS + (int)threadIdx.x; };
    float v[LP_EACH];
    if (a.vec && t0 + LP_TILE <= a.V) {
#pragma unroll
      for (int i = 0; i < LP_EACH / E; i++) {
        const uint4 raw = *reinterpret_cast<const uint4*>(z + index(i * E));
        const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < E; j++)
          v[i * E + j] = __uint_as_float(sizeof(TX) == 4 ? w[j & 3] : j & 1 ? w[j >> 1 & 3] & 0xffff0000u : w[j >> 1 & 3] << 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < LP_EACH; i++) v[i] = index(i) < a.V ? to_float(z[index(i)]) : -INFINITY;
    }
    float m = v[0];
#pragma unroll
    for (int i = 1; i < LP_EACH; i++) m = fmaxf(m, v[i]);
    if (m > sum.m) lp_to(sum, m);
#pragma unroll
    for (int i = 0; i < LP_EACH; i++) {
      const float d = lp_distance(v[i], sum.m), e = __expf(d);
      sum.s += e;
      sum.d = fmaf(d, e, sum.d);
    }
    if (a.top) {
      const bool first = tile == lo;
      if (first) {
        unsigned left = lp_order(m), o = 0;
        for (int i = 0; i * LP_WARPS < a.top; i++) {
          o = __reduce_max_sync(0xffffffffu, left);
          if ((int)__ffs(__ballot_sync(0xffffffffu, left == o)) - 1 == lane) left = 0;
        }
        if (lane == 0) sh.bound[warp] = o;
        __syncthreads();
        o = sh.bound[0];
#pragma unroll
        for (int i = 1; i < LP_WARPS; i++) o = min(o, sh.bound[i]);
        any = o == 0;                                                // (a thread with no number at all: no bound)
        least = any ? 0.f : lp_value(o);
      }
      if (threadIdx.x == 0) sh.joined[(tile + 1) % 3] = 0;           // (its last readers are behind the barrier before the last)
#pragma unroll
      for (int i = 0; i < LP_EACH; i++)
        if (first ? any || v[i] >= least : any || v[i] > least) {
          const unsigned long long key = index(i) < a.V ? lp_key(v[i], index(i)) : 0ull;
          if (key) {
            const int place = n + atomicAdd(&sh.joined[tile % 3], 1);
            if (place < LP_LIST) sh.list[place] = key;
          }
        }
      __syncthreads();
      const int had = n;
      n += sh.joined[tile % 3];
      if (n >= LP_CUT || first) {
        if (n > LP_LIST) {
          // the tile's largest ones, one after the other, in place of those that have joined
          unsigned long long last = ~0ull;
          n = had;
          for (int k = 0; k < a.top; k++) {
            unsigned long long mine = 0;
#pragma unroll
            for (int i = 0; i < LP_EACH; i++) {
              const unsigned long long key = index(i) < a.V ? lp_key(v[i], index(i)) : 0ull;
              if (key < last && key > mine) mine = key;
            }
            mine = lp_warp_max(mine);
            if (lane == 0) sh.best[k & 1][warp] = mine;
            __syncthreads();
            last = sh.best[k & 1][0];
#pragma unroll
            for (int i = 1; i < LP_WARPS; i++) last = max(last, sh.best[k & 1][i]);
            if (!last) break;
            if (threadIdx.x == 0) sh.list[n] = last;
            n++;
          }
        }
        n = lp_cut(sh, n, a.top);
        any = n < a.top;
        least = any ? 0.f : lp_value((unsigned)(sh.list[a.top - 1] >> 32));
      }
    }
  }
  // ---- the CTA's sums
  const float m = lp_value(__reduce_max_sync(0xffffffffu, lp_order(sum.m)));
  lp_to(sum, m);
  sum.s = warp_sum(sum.s);
  sum.d = warp_sum(sum.d);
  if (lane == 0) sh.sum[warp] = sum;
  __syncthreads();
  if (n > a.top) n = lp_cut(sh, n, a.top);
  if (threadIdx.x == 0) {
    sh.n = n;
    LpSum w = sh.sum[0];
    for (int i = 1; i < LP_WARPS; i++) {
      LpSum x = sh.sum[i];
      const float mm = fmaxf(w.m, x.m);
      lp_to(w, mm);
      lp_to(x, mm);
      w.s += x.s;
      w.d += x.d;
    }
    sh.whole = w;
  }
  __syncthreads();
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
      for (int c = 1; c < a.shares; c++) {
        LpSum x;
        const unsigned from = at(&sh.whole, c);
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x.m) : "r"(from) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x.s) : "r"(from + 4) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x.d) : "r"(from + 8) : "memory");
        const float mm = fmaxf(whole.m, x.m);
        lp_to(whole, mm);
        lp_to(x, mm);
        whole.s += x.s;
        whole.d += x.d;
      }
      if (a.top) {
        // every share's list is in order, with at most ``top``: thread (c, i) brings the i-th of share c
        const int c = threadIdx.x >> 5;
        unsigned long long key = 0;
        if (c < a.shares && lane < a.top) {
          int have;
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(have) : "r"(at(&sh.n, c)) : "memory");
          if (lane < have) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(at(&sh.list[lane], c)) : "memory");
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.n = 0;
        __syncthreads();
        if (key) sh.list[atomicAdd(&sh.n, 1)] = key;
        __syncthreads();
        n = lp_cut(sh, sh.n, a.top);
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (share) return;
  }
  const float log_s = logf(whole.s);
  // (a row of minus infinities alone has no probabilities: none is above 0)
  auto log_p = [&](float x) { return whole.s == 0.f ? -INFINITY : x - whole.m - log_s; };
  if (threadIdx.x == 0) {
    const int t = a.tokens[row];
    a.logprob[row] = t >= 0 && t < a.V ? log_p(to_float(z[t])) : __uint_as_float(0x7fc00000u);
    a.entropy[row] = whole.s == 0.f ? 0.f : log_s - whole.d / whole.s;
  }
  if ((int)threadIdx.x < a.top) {
    const bool there = (int)threadIdx.x < n;
    const unsigned long long key = there ? sh.list[threadIdx.x] : 0;
    a.top_ids[(size_t)row * a.top + threadIdx.x] = there ? (int)(0xffffffffu - (unsigned)key) : -1;
    a.top_logprobs[(size_t)row * a.top + threadIdx.x] = there ? log_p(lp_value((unsigned)(key >> 32))) : __uint_as_float(0x7fc00000u);
  }
}

// logits [R, V] float32 or bfloat16, rows ``ld`` elements apart; tokens int32 [R] (outside of [0, V): the log probability NaN); logprob and
// entropy float32 [R]; top_ids int32 and top_logprobs float32 [R, top], top up to 32, of rows with fewer numbers -1 and NaN.
extern "C" int qd_token_logprobs(const void* logits, int dtype, long long ld, const int* tokens, float* logprob, float* entropy,
                                 int* top_ids, float* top_logprobs, int R, int V, int top, int sms, cudaStream_t stream) {
  if (R <= 0) return 0;
  if ((dtype != QD_F32 && dtype != QD_BF16) || V <= 0 || V > (1 << 30) || top < 0 || top > LP_MAX_TOP || top > V || sms < 1)
    return QD_ERR_UNSUPPORTED;
  LpArgs a;
  a.logits = logits; a.tokens = tokens; a.logprob = logprob; a.entropy = entropy; a.top_ids = top_ids; a.top_logprobs = top_logprobs;
  a.R = R; a.V = V; a.top = top; a.ld = ld;
  const int size = dtype == QD_F32 ? 4 : 2;
  a.vec = !((uintptr_t)logits & 15) && ld * size % 16 == 0;
  a.shares = 1;
  while (a.shares < 8 && (long long)R * a.shares * 2 <= 4ll * sms && a.shares * 2 * LP_TILE <= V) a.shares *= 2;
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
