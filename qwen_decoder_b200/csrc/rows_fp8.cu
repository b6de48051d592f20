// Rows into 8 bits (fp8.cuh): as they are, through a gated activation, or through the residual sum's RMS norm.
//
// A warp takes a block of 128 features, four to a lane: the block's largest magnitude is one reduction over the warp (of the bits, which
// order as the magnitudes do), and a lane stores four bytes of a row's 128.  All arithmetic is in float32; the numbers are rounded once,
// to 8 bits.
//
// The reference rounds nothing below 16 bits (its norm and activation: gpu_kernels.cu:32-67, 136-160).
#include "fp8.cuh"

// four neighbouring features, zeros from ``K`` on; ``vec``: they lie on 16 (float32) or 8 bytes (bfloat16)
__device__ __forceinline__ float4 load4(const float* row, int k, int K, bool vec) {
  if (vec && k + 4 <= K) return *reinterpret_cast<const float4*>(row + k);
  return make_float4(k < K ? row[k] : 0.f, k + 1 < K ? row[k + 1] : 0.f, k + 2 < K ? row[k + 2] : 0.f, k + 3 < K ? row[k + 3] : 0.f);
}
__device__ __forceinline__ float4 load4(const bf16* row, int k, int K, bool vec) {
  if (vec && k + 4 <= K) {
    const uint2 raw = *reinterpret_cast<const uint2*>(row + k);
    return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16),
                       __uint_as_float(raw.y & 0xffff0000u));
  }
  return make_float4(k < K ? to_float(row[k]) : 0.f, k + 1 < K ? to_float(row[k + 1]) : 0.f, k + 2 < K ? to_float(row[k + 2]) : 0.f,
                     k + 3 < K ? to_float(row[k + 3]) : 0.f);
}
__device__ __forceinline__ void add4(float4& a, const float4& b) { a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w; }

// A warp's block of 128 features into a row's bytes and its scale's byte; all lanes of the warp
__device__ __forceinline__ void store_block(const float4& v, unsigned char* q_row, unsigned char* s_row, int block, int K) {
  const int lane = threadIdx.x & 31, k = block * FP8_BLOCK + 4 * lane;
  const unsigned m = max(max(fp8_magnitude(v.x), fp8_magnitude(v.y)), max(fp8_magnitude(v.z), fp8_magnitude(v.w)));
  const unsigned byte = fp8_scale_byte(__reduce_max_sync(0xffffffffu, m));
  const float inv = fp8_inverse(byte);
  const unsigned q = fp8_pack4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
  if (k + 4 <= K) *reinterpret_cast<unsigned*>(q_row + k) = q;
  else
    for (int i = 0; i < 4; i++)
      if (k + i < K) q_row[k + i] = (unsigned char)(q >> 8 * i);
  if (lane == 0) s_row[block] = (unsigned char)byte;
}

// ------------------------------------------------------------------------------ rows, and rows of a gated activation
struct RowsArgs {
  const void* x;
  const float* bias;       // of the gate and the up product, [2 K], or null
  unsigned char *q, *s;
  int T, K, blocks, n_parts, act, vec;
  long long ldx, part_stride, ldq, lds;
};

template <typename TX>
__device__ __forceinline__ float4 sum_parts(const RowsArgs& a, const TX* row, int k, int K) {
  float4 v = load4(row, k, K, a.vec);
  for (int p = 1; p < a.n_parts; p++) add4(v, load4(row + p * a.part_stride, k, K, a.vec));
  return v;
}

template <typename TX, bool GATED>
__global__ void __launch_bounds__(256) rows_fp8_kernel(const RowsArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= (long long)a.T * a.blocks) return;
  const int t = (int)(item / a.blocks), block = (int)(item - (long long)t * a.blocks), k = block * FP8_BLOCK + 4 * lane;
  const TX* row = (const TX*)a.x + t * a.ldx;
  float4 v = sum_parts(a, row, k, a.K);
  if (GATED) {
    float4 u = sum_parts(a, row + a.K, k, a.K);
    if (a.bias) {
      add4(v, load4(a.bias, k, a.K, false));
      add4(u, load4(a.bias + a.K, k, a.K, false));
    }
    v.x = fp8_gated(v.x, u.x, a.act);
    v.y = fp8_gated(v.y, u.y, a.act);
    v.z = fp8_gated(v.z, u.z, a.act);
    v.w = fp8_gated(v.w, u.w, a.act);
  }
  store_block(v, a.q + t * a.ldq, a.s + t * a.lds, block, a.K);
}

// q [T, K] e4m3 and s [T, ceil(K / 128)], rows ``ldq`` and ``lds`` bytes apart (a multiple of 4), of
//   gated 0: x [T, K] bfloat16 or float32, rows ``ldx`` apart, or the sum of ``n_parts`` float32 parts ``part_stride`` apart;
//   gated 1: act(g) u, x [T, 2 K]: g and u side by side (or such parts), ``bias`` float32 [2 K] added to their sums, or null.
extern "C" int qd_rows_fp8(const void* x, int dtype, long long ldx, int n_parts, long long part_stride, int gated, int act,
                           const float* bias, void* q, long long ldq, void* s, long long lds, int T, int K, cudaStream_t stream) {
  if (T <= 0 || K <= 0) return 0;
  if ((dtype != QD_F32 && dtype != QD_BF16) || n_parts < 1 || (n_parts > 1 && dtype != QD_F32)) return QD_ERR_UNSUPPORTED;
  if (ldq % 4 || ((uintptr_t)q & 3) || (bias && !gated) || (gated && act != QD_ACT_SILU && act != QD_ACT_GELU_TANH)) return QD_ERR_UNSUPPORTED;
  RowsArgs a;
  a.x = x; a.bias = bias; a.q = (unsigned char*)q; a.s = (unsigned char*)s;
  a.T = T; a.K = K; a.blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK; a.n_parts = n_parts; a.act = act;
  a.ldx = ldx; a.part_stride = part_stride; a.ldq = ldq; a.lds = lds;
  const int bytes = dtype == QD_F32 ? 16 : 8;
  a.vec = !((uintptr_t)x & (bytes - 1)) && ldx % 4 == 0 && part_stride % 4 == 0 && (!gated || K % 4 == 0);
  const long long items = (long long)T * a.blocks;
  if (items > (1ll << 33)) return QD_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)((items + 7) / 8));
#define GO(TX, G) qd_launch(rows_fp8_kernel<TX, G>, grid, dim3(256), 0, stream, a)
  if (gated) { if (dtype == QD_F32) GO(float, true); else GO(bf16, true); }
  else { if (dtype == QD_F32) GO(float, false); else GO(bf16, false); }
#undef GO
  return qd_last_error();
}

// ------------------------------------------------------------------------------ the residual sum's norm
struct NormArgs {
  float* x;
  const void* delta;
  const float *dscale, *w;
  unsigned char *q, *s;
  const int* rows;
  int D, blocks, n_parts, write_back, vec;
  float eps;
  long long part_stride, ldq, lds;
};

// One CTA to a row.  A warp holds up to VPT of the row's blocks in registers.
template <typename TD, int VPT>
__global__ void __launch_bounds__(1024) norm_fp8_kernel(const NormArgs a) {
  __shared__ float scratch[40];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x;
  const size_t at = (size_t)(a.rows ? a.rows[r] : r) * a.D;
  float4 v[VPT];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const int block = warp + i * warps, k = block * FP8_BLOCK + 4 * lane;
    v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (block < a.blocks) {
      v[i] = load4(a.x + at, k, a.D, a.vec);
      if (a.delta) {
        const TD* dp = (const TD*)a.delta + at;
        float4 d = load4(dp, k, a.D, a.vec);
        for (int p = 1; p < a.n_parts; p++) add4(d, load4(dp + p * a.part_stride, k, a.D, a.vec));
        if (a.dscale) {
          const float4 f = load4(a.dscale, k, a.D, a.vec);
          d.x *= f.x; d.y *= f.y; d.z *= f.z; d.w *= f.w;
        }
        add4(v[i], d);
        if (a.write_back) {
          float* to = a.x + at + k;
          if (a.vec && k + 4 <= a.D) *reinterpret_cast<float4*>(to) = v[i];
          else {
            if (k < a.D) to[0] = v[i].x;
            if (k + 1 < a.D) to[1] = v[i].y;
            if (k + 2 < a.D) to[2] = v[i].z;
            if (k + 3 < a.D) to[3] = v[i].w;
          }
        }
      }
      ss += v[i].x * v[i].x + v[i].y * v[i].y + v[i].z * v[i].z + v[i].w * v[i].w;
    }
  }
  ss = block_sum(ss, scratch);
  const float inv = 1.0f / sqrtf(ss / (float)a.D + a.eps);
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const int block = warp + i * warps, k = block * FP8_BLOCK + 4 * lane;
    if (block < a.blocks) {
      const float4 w = load4(a.w, k, a.D, a.vec);
      v[i].x = v[i].x * inv * w.x; v[i].y = v[i].y * inv * w.y; v[i].z = v[i].z * inv * w.z; v[i].w = v[i].w * inv * w.w;
      store_block(v[i], a.q + (size_t)r * a.ldq, a.s + (size_t)r * a.lds, block, a.D);
    }
  }
}

// x [.., D] float32 += delta (bfloat16 or float32, or the sum of ``n_parts`` float32 parts ``part_stride`` apart; times ``dscale`` [D] if
// given; null: nothing to add) in the rows that ``rows`` names (null: all n_rows), kept where ``write_back``; q and s: that row's
// x / sqrt(mean(x^2) + eps) * w in 8 bits.
extern "C" int qd_add_rmsnorm_fp8(float* x, const void* delta, int delta_dtype, const float* dscale, const float* w, void* q,
                                  long long ldq, void* s, long long lds, const int* rows, int n_rows, int D, float eps, int write_back,
                                  int n_parts, long long part_stride, cudaStream_t stream) {
  if (n_rows <= 0 || D <= 0) return 0;
  if (delta && delta_dtype != QD_BF16 && delta_dtype != QD_F32) return QD_ERR_UNSUPPORTED;
  if (n_parts < 1 || (n_parts > 1 && delta_dtype != QD_F32) || ldq % 4 || ((uintptr_t)q & 3)) return QD_ERR_UNSUPPORTED;
  NormArgs a;
  a.x = x; a.delta = delta; a.dscale = dscale; a.w = w; a.q = (unsigned char*)q; a.s = (unsigned char*)s; a.rows = rows;
  a.D = D; a.blocks = (D + FP8_BLOCK - 1) / FP8_BLOCK; a.n_parts = n_parts; a.write_back = write_back; a.eps = eps;
  a.part_stride = part_stride; a.ldq = ldq; a.lds = lds;
  a.vec = D % 4 == 0 && part_stride % 4 == 0 && !(((uintptr_t)x | (uintptr_t)w | (uintptr_t)dscale) & 15) &&
          !((uintptr_t)delta & (delta_dtype == QD_BF16 ? 7 : 15));
  if (a.blocks > 32 * 16) return QD_ERR_UNSUPPORTED;       // 65,536 features
  const int vpt = a.blocks <= 32 ? 1 : a.blocks <= 64 ? 2 : a.blocks <= 128 ? 4 : 16;
  const dim3 grid(n_rows), block(32 * ((a.blocks + vpt - 1) / vpt));
#define GO(TD, V) qd_launch(norm_fp8_kernel<TD, V>, grid, block, 0, stream, a)
#define PICK(TD) do { if (vpt == 1) GO(TD, 1); else if (vpt == 2) GO(TD, 2); else if (vpt == 4) GO(TD, 4); else GO(TD, 16); } while (0)
  if (delta && delta_dtype == QD_BF16) PICK(bf16); else PICK(float);
#undef PICK
#undef GO
  return qd_last_error();
}
