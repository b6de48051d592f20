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
// logits the lowest index is the largest key.  Every warp keeps a list of keys in shared memory and a threshold that at least ``top`` logits
// of the list reach; only larger ones join it (a warp's later tiles have higher indices: equal ones lose), and it is cut back to its first
// ``top`` when it has LP_CUT: no barrier of the CTA holds the reading up (with one list to a CTA and a barrier to every tile 509 rows of
// 152,064 took 80 us, without a list 52).  For the first tile the threshold is the ``top``-th of the lanes' maxima.  Where a tile brings more
// than the list holds (rows in rising order, a thousand equal logits), its largest ``top`` are taken one by one.  Of L sorted lists the
// keys that count are those not below the least of the lists' ceil(top / L)-th keys, which ``top`` keys reach: few, and put in order by
// counting for each how many are larger.
//
// The reference has no log probabilities; its sampler's softmax is common.cpp:576-629.
#include "common.cuh"

#define LP_THREADS 256
#define LP_WARPS (LP_THREADS / 32)
#define LP_EACH 16                           // logits of a thread's tile
#define LP_TILE (LP_THREADS * LP_EACH)
#define LP_MAX_TOP 32
#define LP_LIST 96                           // of a warp
#define LP_CUT 64
#define LP_MAX_SHARES 16
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
  unsigned long long list[LP_WARPS][LP_LIST], joined[LP_MAX_SHARES * LP_MAX_TOP], sorted[LP_MAX_TOP];
  LpSum sum[LP_WARPS], whole;
  int n[LP_WARPS], n_joined, n_sorted;
};

// A warp's list of ``n`` keys in order, cut to the first ``top``; their number
__device__ __forceinline__ int lp_cut(unsigned long long* list, int n, int top) {
  const int lane = threadIdx.x & 31;
  unsigned long long mine[LP_LIST / 32];
  int before[LP_LIST / 32];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < LP_LIST / 32; i++) {
    mine[i] = lane + 32 * i < n ? list[lane + 32 * i] : 0ull;
    before[i] = 0;
  }
#pragma unroll 4
  for (int j = 0; j < n; j++) {
    const unsigned long long k = list[j];
#pragma unroll
    for (int i = 0; i < LP_LIST / 32; i++) before[i] += k > mine[i];
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < LP_LIST / 32; i++)
    if (mine[i] && before[i] < top) list[before[i]] = mine[i];
  __syncwarp();
  return min(n, top);
}

template <typename TX>
__global__ void __launch_bounds__(LP_THREADS, 4) logprobs_kernel(const LpArgs a) {
  __shared__ LpShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x / a.shares, share = blockIdx.x - row * a.shares;
  unsigned long long* list = sh.list[warp];
  if (threadIdx.x == 0) sh.n_joined = 0;
  pdl_launch_dependents();
  pdl_wait();
  const TX* z = (const TX*)a.logits + row * a.ld;
  const int tiles = (a.V + LP_TILE - 1) / LP_TILE;
  const int lo = (int)((long long)tiles * share / a.shares), hi = (int)((long long)tiles * (share + 1) / a.shares);
  constexpr int E = 16 / (int)sizeof(TX);                            // of a load
  LpSum sum = {LP_LOWEST, 0.f, 0.f};
  float least = 0.f;                                                 // a logit joins the warp's list above this, ...
  bool any = true;                                                   // ... or any does
  int n = 0;                                                         // of the list, the same to all lanes
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
      const float d = (v[i] - sum.m) * LP_LOG2E, e = lp_exp2(d);
      sum.s += e;                                                    // (NaN comes this way)
      sum.d = fmaf(fmaxf(d, -256.f), e, sum.d);
    }
    if (!a.top) continue;
    const bool first = tile == lo;
    if (first) {
      unsigned left = lp_order(m), o = 0;
      for (int i = 0; i < a.top; i++) {
        o = __reduce_max_sync(0xffffffffu, left);
        if ((int)__ffs(__ballot_sync(0xffffffffu, left == o)) - 1 == lane) left = 0;
      }
      any = o == 0;                                                  // (a lane with no number at all: no bound)
      least = any ? 0.f : lp_value(o);
    }
    if (!__any_sync(0xffffffffu, any || m > least || (first && m == least))) continue;
    unsigned hits = 0;
    int more = 0;
    auto count = [&]() {
      hits = 0;
#pragma unroll
      for (int i = 0; i < LP_EACH; i++)
        if ((any ? v[i] == v[i] : v[i] > least || (first && v[i] == least)) && index(i) < a.V) hits |= 1u << i;
      more = __reduce_add_sync(0xffffffffu, __popc(hits));
    };
    auto cut = [&]() {
      n = lp_cut(list, n, a.top);
      any = n < a.top;
      least = any ? 0.f : lp_value((unsigned)(list[a.top - 1] >> 32));
    };
    count();
    if (n + more > LP_LIST && n > a.top) {
      cut();
      count();
    }
    if (n + more > LP_LIST) {
      // the tile's largest ones, one after the other
      unsigned long long last = ~0ull;
      for (int k = 0; k < a.top; k++) {
        unsigned long long mine = 0;
#pragma unroll 1
        for (int i = 0; i < LP_EACH; i++) {                          // (read again: kept numbers would cost every tile registers)
          const int at = index(i);
          const unsigned long long key = at < a.V ? lp_key(to_float(z[at]), at) : 0ull;
          if (key < last && key > mine) mine = key;
        }
        last = lp_warp_max(mine);
        if (!last) break;
        if (lane == 0) list[n] = last;
        n++;
      }
      cut();
    } else {
      int at = __popc(hits);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += x;
      }
      at += n - __popc(hits);
#pragma unroll
      for (int i = 0; i < LP_EACH; i++)
        if (hits >> i & 1) list[at++] = lp_key(v[i], index(i));
      n += more;
      if (n >= LP_CUT || first) cut();
    }
  }
  // ---- the CTA's sums and its list
  const float m = lp_value(__reduce_max_sync(0xffffffffu, lp_order(sum.m)));
  lp_to(sum, m);
  sum.s = warp_sum(sum.s);
  sum.d = warp_sum(sum.d);
  if (a.top) n = lp_cut(list, n, a.top);
  if (lane == 0) {
    sh.sum[warp] = sum;
    sh.n[warp] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    LpSum w = sh.sum[0];
    for (int i = 1; i < LP_WARPS; i++) lp_join(w, sh.sum[i]);
    sh.whole = w;
  }
  // keys of sorted lists that are not below ``least`` (of the lists' ``nth`` keys, 0 where one has fewer) join, and are put in order
  auto order = [&]() {
    __syncthreads();
    const int total = sh.n_joined;
    for (int i = threadIdx.x; i < total; i += LP_THREADS) {
      const unsigned long long mine = sh.joined[i];
      int before = 0;
      for (int j = 0; j < total; j++) before += sh.joined[j] > mine;
      if (before < a.top) sh.sorted[before] = mine;
    }
    if (threadIdx.x == 0) sh.n_sorted = min(total, a.top);
    __syncthreads();
  };
  if (a.top) {
    const int nth = (a.top + LP_WARPS - 1) / LP_WARPS - 1;
    unsigned long long bound = ~0ull;
#pragma unroll
    for (int i = 0; i < LP_WARPS; i++) bound = min(bound, nth < sh.n[i] ? sh.list[i][nth] : 0ull);
    if (lane < n && list[lane] >= bound) sh.joined[atomicAdd(&sh.n_joined, 1)] = list[lane];
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
      // (a lane to a share: all of their words are on their way together)
      unsigned long long nth_key = 0;
      int have = 0;
      if (warp == 0 && lane < a.shares) {
        LpSum x;
        const unsigned from = at(&sh.whole, lane);
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x.m) : "r"(from) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x.s) : "r"(from + 4) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x.d) : "r"(from + 8) : "memory");
        sum = x;
      }
      if (warp == 0) {
        if (lane >= a.shares) sum = {LP_LOWEST, 0.f, 0.f};
        lp_to(sum, lp_value(__reduce_max_sync(0xffffffffu, lp_order(sum.m))));
        whole.m = sum.m;
        whole.s = warp_sum(sum.s);
        whole.d = warp_sum(sum.d);
      }
      if (a.top) {
        const int nth = (a.top + a.shares - 1) / a.shares - 1;
        if (lane < a.shares) {
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(have) : "r"(at(&sh.n_sorted, lane)) : "memory");
          asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(nth_key) : "r"(at(&sh.sorted[nth], lane)) : "memory");
          if (nth >= have) nth_key = 0;
        } else {
          nth_key = ~0ull;
        }
        const unsigned long long bound = ~lp_warp_max(~nth_key);
        // warp w brings the lists of shares w, w + 8
        unsigned long long key[LP_MAX_SHARES / LP_WARPS];
#pragma unroll
        for (int i = 0; i < LP_MAX_SHARES / LP_WARPS; i++) {
          const int c = warp + i * LP_WARPS, its = __shfl_sync(0xffffffffu, have, c & 31);
          key[i] = 0;
          if (c < a.shares && lane < its) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key[i]) : "r"(at(&sh.sorted[lane], c)) : "memory");
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.n_joined = 0;
        __syncthreads();
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
  n = a.top ? sh.n_sorted : 0;
  const float log_s = logf(whole.s);
  // (a row of minus infinities alone has no probabilities: none is above 0)
  auto log_p = [&](float x) { return whole.s == 0.f ? -INFINITY : x - whole.m - log_s; };
  if (threadIdx.x == 0) {
    const int t = a.tokens[row];
    a.logprob[row] = t >= 0 && t < a.V ? log_p(to_float(z[t])) : __uint_as_float(0x7fc00000u);
    a.entropy[row] = whole.s == 0.f ? 0.f : log_s - LP_LN2 * (whole.d / whole.s);
  }
  if ((int)threadIdx.x < a.top) {
    const bool there = (int)threadIdx.x < n;
    const unsigned long long key = there ? sh.sorted[threadIdx.x] : 0;
    a.top_ids[(size_t)row * a.top + threadIdx.x] = there ? (int)(0xffffffffu - (unsigned)key) : -1;
    a.top_logprobs[(size_t)row * a.top + threadIdx.x] = there ? log_p(lp_value((unsigned)(key >> 32))) : __uint_as_float(0x7fc00000u);
  }
}

// logits [R, V] float32 or bfloat16, rows ``ld`` elements apart; tokens int32 [R] (outside of [0, V): the log probability NaN); logprob and
// entropy float32 [R]; top_ids int32 and top_logprobs float32 [R, top], top up to 32, of rows with fewer numbers -1 and NaN.
extern "C" int qd_token_logprobs(const void* logits, int dtype, long long ld, const int* tokens, float* logprob, float* entropy,
                                 int* top_ids, float* top_logprobs, int R, int V, int top, int sms, int shares, cudaStream_t stream) {
  if (R <= 0) return 0;
  if ((dtype != QD_F32 && dtype != QD_BF16) || V <= 0 || V > (1 << 30) || top < 0 || top > LP_MAX_TOP || top > V || sms < 1 || shares > LP_MAX_SHARES)
    return QD_ERR_UNSUPPORTED;
  LpArgs a;
  a.logits = logits; a.tokens = tokens; a.logprob = logprob; a.entropy = entropy; a.top_ids = top_ids; a.top_logprobs = top_logprobs;
  a.R = R; a.V = V; a.top = top; a.ld = ld;
  const int size = dtype == QD_F32 ? 4 : 2;
  a.vec = !((uintptr_t)logits & 15) && ld * size % 16 == 0;
  a.shares = shares > 0 ? shares : 1;
  while (shares <= 0 && a.shares < LP_MAX_SHARES && (long long)R * a.shares * 2 <= 4ll * sms && a.shares * 2 * LP_TILE <= V) a.shares *= 2;
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
  if (dtype == QD_F32) cudaLaunchKernelEx(&cfg, logprobs_kernel<float>, a);
  else cudaLaunchKernelEx(&cfg, logprobs_kernel<bf16>, a);
  return qd_last_error();
}
