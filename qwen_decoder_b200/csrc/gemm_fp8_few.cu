// Contraction Y[T, N] = X[T, K] * W[N, K]^T of rows in 8 bits (fp8.cuh) for up to 16 tokens: bound by reading W once.
//
// A warp goes through blocks of 16 rows of W by 128 of k, each 2 KB, which travel into its own part of shared memory by asynchronous copies
// of 16 bytes, some blocks ahead, the first of them before the kernel before this one has ended, and the tokens' 128 of k with them.  A lane
// reads back what it has copied itself: no barrier stands between the copies and the products.  (With the tokens loaded where they are needed
// 151,936 x 2,048 took 104 us for 8 of them.)  mma.sync m16n8k32 (W's rows the 16, tokens the 8) sums a block; the
// block's scales, powers of two, are factors of its sums, which go on in float32.  The four bytes that an operand's register holds
// are any four of k as long as both operands hold the same: a lane takes 16 neighbouring bytes twice, not four times four.  The warps of a
// CTA, and with few rows the CTAs of a cluster, share the blocks of 16 rows' K and add their sums up over shared memory, in their order.
//
// What bounds it: a multiprocessor's 60 clocks to a block for the MMAs and as many for the rest, 4 TB/s; the product on tcgen05
// (gemm_fp8.cu) reads large matrices at 6 TB/s but has a longer way through barriers, tensor memory and a cluster's joining.  Measured
// here / there, us, in captured graphs, 1 and 16 tokens:
//   2,048 x 2,048    3.4 /  4.9    4.2 / 5.1       3,584 x 3,584    5.1 /  6.7    7.0 /  7.0
//   2,560 x 2,048    3.5 /  5.1    4.5 / 5.4       4,608 x 3,584    5.8 /  7.3    7.3 /  7.5
//   2,048 x 5,120    5.3 /  6.7    7.3 / 6.9       2,048 x 11,008   8.6 /  9.1   11.8 /  9.4
//   1,000 x 1,000    2.1 /  4.1    2.6 / 4.3      22,016 x 2,048   13.1 / 10.3   19.2 / 11.3
//
// The reference has 16-bit products only (cublasHgemm, gpu_kernels.cu:431-436).
#include "entry_points.h"
#include "fp8.cuh"

#define FW_WARPS 8
#define FW_ROWS 16
// blocks under way to a warp, and their bytes with those of NT times 8 tokens: 96 KB to a CTA, two CTAs to a multiprocessor
template <int NT> struct FwRing {
  static constexpr int DEPTH = NT == 1 ? 4 : 3, BYTES = (FW_ROWS + 8 * NT) * FP8_BLOCK, ALL = FW_WARPS * DEPTH * BYTES;
};
#define FW_STRIDE (FW_ROWS + 1)              // of a token's sums in shared memory

struct FwParams {
  const unsigned char *w, *sw, *x, *sx;
  long long ldw, ldsw, ldx, ldsx, ldo;
  const float* bias;
  void* out;
  int T, N, K, blocks, tiles, shares;      // CTAs that share a tile's K
  int resident;                            // no kernel before this one writes W or its scales
};

// 16 bytes, of which ``there`` (0 to 16) come from memory and the others are zero
__device__ __forceinline__ void fw_copy(unsigned to, const unsigned char* from, int there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there) : "memory");
}
__device__ __forceinline__ float fw_scale(unsigned byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : byte ? byte << 23 : 0x00400000u);
}
__device__ __forceinline__ void fw_mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: groups of 8 tokens; SHARED: a tile's K belongs to the CTAs of a cluster
template <int NT, typename TO, bool SHARED>
__global__ void __launch_bounds__(FW_WARPS * 32, 2) gemm_fp8_few_kernel(const FwParams p) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float sums[2][FW_WARPS][NT * 8 * FW_STRIDE];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int shares = SHARED ? p.shares : 1, share = SHARED ? blockIdx.x % shares : 0;
  const int worker = SHARED ? blockIdx.x / shares : blockIdx.x, workers = SHARED ? gridDim.x / shares : gridDim.x;
  const int b0 = p.blocks * share / shares + warp, b1 = p.blocks * (share + 1) / shares;       // this warp's first block, the CTA's end
  pdl_launch_dependents();
  constexpr int DEPTH = FwRing<NT>::DEPTH, BYTES = FwRing<NT>::BYTES;
  unsigned char* mine = ring + warp * DEPTH * BYTES + lane * 16;
  const unsigned mine_at = (unsigned)__cvta_generic_to_shared(mine);
  // a row's two pieces of a block into its place in a slot
  auto piece = [&](int slot, int place, const unsigned char* row, bool there, int k) {
    const unsigned to = mine_at + slot * BYTES + place * 1024;
    const int left = there ? p.K - k : 0;
    fw_copy(to, row + (left > 0 ? k : 0), max(0, min(16, left)));
    fw_copy(to + 512, row + (left > 64 ? k + 64 : 0), max(0, min(16, left - 64)));
  };
  auto weights = [&](int slot, int tile, int b) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int row = tile * FW_ROWS + g + 8 * i;
      piece(slot, i, p.w + (row < p.N ? row : 0) * p.ldw, row < p.N, b * FP8_BLOCK + 16 * t);
    }
  };
  auto tokens = [&](int slot, int b) {
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const int token = 8 * j + g;
      piece(slot, 2 + j, p.x + (token < p.T ? token : 0) * p.ldx, token < p.T, b * FP8_BLOCK + 16 * t);
    }
  };
  // a place in a warp's sequence of (tile, block)
  struct Place { int tile, b; };
  auto next = [&](Place& q) {
    q.b += FW_WARPS;
    if (q.b >= b1) {
      q.b = b0;
      q.tile += workers;
    }
  };
  auto commit = [&]() { asm volatile("cp.async.commit_group;" ::: "memory"); };
  const Place first = {b0 < b1 ? worker : p.tiles, b0};       // (a warp without blocks asks for none)
  Place ask = first;
  if (!p.resident) pdl_wait();
#pragma unroll 1
  for (int i = 0; i < DEPTH; i++) {
    if (ask.tile < p.tiles) {
      weights(i, ask.tile, ask.b);
      next(ask);
    }
    commit();
  }
  pdl_wait();
  Place x = first;
#pragma unroll 1
  for (int i = 0; i < DEPTH; i++) {
    if (x.tile < p.tiles) {
      tokens(i, x.b);
      next(x);
    }
    commit();
  }
  // the next block's scales, as they lie in memory
  unsigned char sw[2], sx[NT][2];
  Place scales = first;
  auto load_scales = [&]() {
    if (scales.tile >= p.tiles) return;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int row = scales.tile * FW_ROWS + g + 8 * i;
      sw[i] = row < p.N ? p.sw[row * p.ldsw + scales.b] : 0;
    }
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int c = 8 * j + 2 * t + i;
        sx[j][i] = c < p.T ? p.sx[c * p.ldsx + scales.b] : 0;
      }
    next(scales);
  };
  load_scales();
  int slot = 0, n = 0;
  for (int tile = worker; tile < p.tiles; tile += workers, n++) {
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    for (int b = b0; b < b1; b += FW_WARPS) {
      const float s0 = fw_scale(sw[0]), s1 = fw_scale(sw[1]);
      float c[NT][2];
#pragma unroll
      for (int j = 0; j < NT; j++) {
        c[j][0] = fw_scale(sx[j][0]);
        c[j][1] = fw_scale(sx[j][1]);
      }
      load_scales();
      asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
      const uint4* from = reinterpret_cast<const uint4*>(mine + slot * BYTES);
      const uint4 a0 = from[0], a1 = from[32], e0 = from[64], e1 = from[96];     // rows g and g + 8, two pieces each
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const uint4 lo = from[128 + 64 * j], hi = from[160 + 64 * j];
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        fw_mma(v, a0.x, e0.x, a0.y, e0.y, lo.x, lo.y);
        fw_mma(v, a0.z, e0.z, a0.w, e0.w, lo.z, lo.w);
        fw_mma(v, a1.x, e1.x, a1.y, e1.y, hi.x, hi.y);
        fw_mma(v, a1.z, e1.z, a1.w, e1.w, hi.z, hi.w);
        acc[j][0] = fmaf(v[0] * s0, c[j][0], acc[j][0]);
        acc[j][1] = fmaf(v[1] * s0, c[j][1], acc[j][1]);
        acc[j][2] = fmaf(v[2] * s1, c[j][0], acc[j][2]);
        acc[j][3] = fmaf(v[3] * s1, c[j][1], acc[j][3]);
      }
      if (ask.tile < p.tiles) {
        weights(slot, ask.tile, ask.b);
        tokens(slot, ask.b);
        next(ask);
      }
      commit();
      if (++slot == DEPTH) slot = 0;
    }
    float* to = sums[n & 1][warp];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int i = 0; i < 4; i++) to[(8 * j + 2 * t + (i & 1)) * FW_STRIDE + g + 8 * (i >> 1)] = acc[j][i];
    if (!SHARED) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    // (with a cluster every CTA adds up its part of the tile's numbers)
    const int all = NT * 8 * FW_ROWS;
    for (int e = all * share / shares + threadIdx.x; e < all * (share + 1) / shares; e += FW_WARPS * 32) {
      const int token = e / FW_ROWS, row = e % FW_ROWS, f = tile * FW_ROWS + row;
      if (token < p.T && f < p.N) {
        float s = p.bias ? p.bias[f] : 0.f;
        if (!SHARED) {
#pragma unroll
          for (int i = 0; i < FW_WARPS; i++) s += sums[n & 1][i][token * FW_STRIDE + row];
        } else {
          for (int c = 0; c < shares; c++) {
            float v[FW_WARPS];
#pragma unroll
            for (int i = 0; i < FW_WARPS; i++) {
              unsigned at;
              asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at)
                           : "r"((unsigned)__cvta_generic_to_shared(&sums[n & 1][i][token * FW_STRIDE + row])), "r"(c));
              asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[i]) : "r"(at) : "memory");
            }
#pragma unroll
            for (int i = 0; i < FW_WARPS; i++) s += v[i];
          }
        }
        ((TO*)p.out)[token * p.ldo + f] = from_float<TO>(s);
      }
    }
  }
  // (the others may still read this CTA's sums)
  if (SHARED) asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int NT, typename TO, bool SHARED>
static int fw_launch(const FwParams& p, int ctas, cudaStream_t stream) {
  static bool allowed[64];                     // by device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return QD_ERR_UNSUPPORTED;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(gemm_fp8_few_kernel<NT, TO, SHARED>, cudaFuncAttributeMaxDynamicSharedMemorySize, FwRing<NT>::ALL) != cudaSuccess)
      return (int)cudaGetLastError();
    allowed[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(FW_WARPS * 32);
  cfg.dynamicSmemBytes = FwRing<NT>::ALL;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.shares;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = qd_pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&cfg, gemm_fp8_few_kernel<NT, TO, SHARED>, p);
  return qd_last_error();
}

// Few tiles of a long K: K shared by as many CTAs as run beside one another, two to a multiprocessor, two blocks to a warp at least
// (us with 1, 2 and 4 of them: 2,048 x 11,008 12.8, 8.6 and 9.9, 2,048 x 2,048 3.1, 3.7 and 5.4, 200 x 12,000 8.9, 5.8 and 4.3); else the
// tiles evenly over these, in rounds.
struct FwCut { int blocks, tiles, shares, rounds; };
static FwCut fw_cut(int N, int K, int sms) {
  const int most = 2 * sms;
  FwCut c = {(K + FP8_BLOCK - 1) / FP8_BLOCK, (N + FW_ROWS - 1) / FW_ROWS, 1, 0};
  while (c.shares < 8 && c.tiles * c.shares * 2 <= most && c.blocks >= c.shares * 4 * FW_WARPS) c.shares *= 2;
  c.rounds = (c.tiles * c.shares + most - 1) / most;
  return c;
}

// Whether this kernel is the faster one for T tokens, or the one on tcgen05 is.  Its time goes by the steps that a CTA makes one after the other, each a
// block to each of its warps, and an end to each tile; the other's by bytes, from 4 us on.  Measured in captured graphs at 274 sizes of 0.5 to
// 50 MB, K 256 to 18,944, with 1 to 16 tokens, us less here on average:
//   steps                1     2     3     4     5     6     7     8    10
//   up to 8 tokens      1.7   1.4   1.4   0.7   0.0  -0.4  -1.2  -1.3  -2.9
//   9 to 16             1.4   0.6   0.0  -0.9  -1.9  -2.9  -4.0  -4.6  -6.9
// Between other launches it is ahead by 1 to 4 us more (the other's code has to be fetched again): among the layers of ten widths, products of up
// to 6 steps and 8 tokens took 1.0 to 6.5 us less here, of up to 4 steps and 16 tokens 0.7 to 4.7 less but for two (0.6 and 1.1 more), of 5
// and more steps and 16 tokens 0.9 to 21 more.  In a graph of nothing else the rule's choices take 0.5 % longer than the best of both up to 8
// tokens, 1.3 % up to 16.
extern "C" int qd_gemm_fp8_few_wanted(int T, int N, int K, int sms) {
  if (T > QD_FP8_FEW_TOKENS || N > (1 << 30) || K <= 0 || K > (1 << 30) || sms < 1) return 0;
  const FwCut c = fw_cut(N, K, sms);
  const long long steps = ((c.blocks + c.shares - 1) / c.shares + FW_WARPS - 1) / FW_WARPS, all = c.rounds * (steps + 1);
  return T <= 8 ? all <= 7 : all + (c.shares > 1) <= 5;
}

// X [T, K] and W [N, K] e4m3, rows ``ldx`` and ``ldw`` bytes apart (multiples of 16, as the addresses), with scales sx and sw, rows ``ldsx``
// and ``ldsw`` bytes apart; out [T, N] = X W^T (+ bias float32 [N]), bfloat16 or float32, rows ``ldo`` apart.  T up to 16.
// ``resident``: W and sw are written by nothing that may still run on the stream (they are asked for before that has ended).
extern "C" int qd_gemm_fp8_few(const void* W, long long ldw, const void* sw, long long ldsw, const void* X, long long ldx, const void* sx,
                               long long ldsx, const float* bias, void* out, int out_dtype, long long ldo, int T, int N, int K, int resident,
                               int sms, cudaStream_t stream) {
  if (T <= 0 || N <= 0) return 0;
  if (T > QD_FP8_FEW_TOKENS || N > (1 << 30) || K <= 0 || K > (1 << 30) || ldx % 16 || ldw % 16 || ldx < K || ldw < K || ((((uintptr_t)W | (uintptr_t)X) & 15)) ||
      sms < 1 || !out)
    return QD_ERR_UNSUPPORTED;
  FwParams p;
  p.w = (const unsigned char*)W; p.sw = (const unsigned char*)sw; p.x = (const unsigned char*)X; p.sx = (const unsigned char*)sx;
  p.ldw = ldw; p.ldsw = ldsw; p.ldx = ldx; p.ldsx = ldsx; p.ldo = ldo; p.bias = bias; p.out = out;
  p.T = T; p.N = N; p.K = K; p.resident = resident;
  const FwCut c = fw_cut(N, K, sms);
  p.blocks = c.blocks; p.tiles = c.tiles; p.shares = c.shares;
  if (ldsx < p.blocks || ldsw < p.blocks) return QD_ERR_UNSUPPORTED;
  const int workers = (c.tiles + c.rounds - 1) / c.rounds, ctas = workers * c.shares;
#define GO(NT, TO) return p.shares > 1 ? fw_launch<NT, TO, true>(p, ctas, stream) : fw_launch<NT, TO, false>(p, ctas, stream)
  if (out_dtype == QD_BF16) { if (T <= 8) GO(1, bf16); else GO(2, bf16); }
  if (out_dtype == QD_F32) { if (T <= 8) GO(1, float); else GO(2, float); }
#undef GO
  return QD_ERR_UNSUPPORTED;
}
