// Rows into 8 bits (fp8.cuh): as they are, through a gated activation, or through the residual sum's RMS norm.
//
// A warp takes a block of 128 features, four to a lane: the block's largest magnitude is one reduction over the warp (of the bits, which
// order as the magnitudes do), and a lane stores four bytes of a row's 128.  All arithmetic is in float32; the numbers are rounded once,
// to 8 bits.
//
// The reference rounds nothing below 16 bits (its norm and activation: gpu_kernels.cu:32-67, 136-160).
#include "entry_points.h"
#include "fp8.cuh"

// Four neighbouring features, zeros from ``K`` on.  VEC: K is a multiple of 4 and they lie on 16 (float32) or 8 bytes (bfloat16): one
// load behind a predicate, of which as many are under way at a time as a thread has room for.
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* row, int k, int K) {
  if (VEC) return k < K ? *reinterpret_cast<const float4*>(row + k) : make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(k < K ? row[k] : 0.f, k + 1 < K ? row[k + 1] : 0.f, k + 2 < K ? row[k + 2] : 0.f, k + 3 < K ? row[k + 3] : 0.f);
}
template <bool VEC>
__device__ __forceinline__ float4 load4(const bf16* row, int k, int K) {
  if (VEC) {
    const uint2 raw = k < K ? *reinterpret_cast<const uint2*>(row + k) : make_uint2(0, 0);
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
  int T, K, blocks, n_parts, act;
  long long ldx, part_stride, ldq, lds;
};

// A warp's EACH blocks, four features to a lane of each, of the sum of a row's parts in their order, four parts' loads together
template <bool VEC, int EACH, typename TX>
__device__ __forceinline__ void sum_parts(float4 (&v)[EACH], const TX* row, int k0, int step, int K, int n_parts, long long part_stride) {
#pragma unroll
  for (int i = 0; i < EACH; i++) v[i] = load4<VEC>(row, k0 + i * step, K);
  if (sizeof(TX) == 2) return;
  for (int p0 = 1; p0 < n_parts; p0 += 4) {
    float4 d[4][EACH];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int i = 0; i < EACH; i++) d[j][i] = load4<VEC>(row + (p0 + j) * part_stride, k0 + i * step, p0 + j < n_parts ? K : 0);
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int i = 0; i < EACH; i++) add4(v[i], d[j][i]);
  }
}

// A warp takes EACH neighbouring blocks of a row, all of their loads before the first is used
template <typename TX, bool GATED, int EACH, bool VEC>
__global__ void __launch_bounds__(256) rows_fp8_kernel(const RowsArgs a) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, runs = (a.blocks + EACH - 1) / EACH;
  const unsigned item = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = item / runs, b0 = (item - t * runs) * EACH, k0 = b0 * FP8_BLOCK + 4 * lane;
  if (t >= a.T) return;
  const TX* row = (const TX*)a.x + t * a.ldx;
  pdl_wait();
  float4 v[EACH], u[EACH];
  sum_parts<VEC>(v, row, k0, FP8_BLOCK, a.K, a.n_parts, a.part_stride);
  if (GATED) sum_parts<VEC>(u, row + a.K, k0, FP8_BLOCK, a.K, a.n_parts, a.part_stride);
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    if (b0 + i >= a.blocks) break;
    if (GATED) {
      if (a.bias) {
        add4(v[i], load4<false>(a.bias, k0 + i * FP8_BLOCK, a.K));
        add4(u[i], load4<false>(a.bias + a.K, k0 + i * FP8_BLOCK, a.K));
      }
      v[i].x = fp8_gated(v[i].x, u[i].x, a.act);
      v[i].y = fp8_gated(v[i].y, u[i].y, a.act);
      v[i].z = fp8_gated(v[i].z, u[i].z, a.act);
      v[i].w = fp8_gated(v[i].w, u[i].w, a.act);
    }
    store_block(v[i], a.q + t * a.ldq, a.s + t * a.lds, b0 + i, a.K);
  }
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
  const bool vec = !((uintptr_t)x & (bytes - 1)) && ldx % 4 == 0 && part_stride % 4 == 0 && K % 4 == 0;
  // few blocks: one to a warp, over as many multiprocessors as there are; many: four, for more bytes on their way
  const int each = (long long)T * a.blocks > 4096 ? 4 : 1;
  const long long items = (long long)T * ((a.blocks + each - 1) / each);
  if (items > (1ll << 31)) return QD_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)((items + 7) / 8));
#define GO2(TX, G, V) do { if (each == 4) qd_launch(rows_fp8_kernel<TX, G, 4, V>, grid, dim3(256), 0, stream, a);             \
                           else qd_launch(rows_fp8_kernel<TX, G, 1, V>, grid, dim3(256), 0, stream, a); } while (0)
#define GO(TX, G) do { if (vec) GO2(TX, G, true); else GO2(TX, G, false); } while (0)
  if (gated) { if (dtype == QD_F32) GO(float, true); else GO(bf16, true); }
  else { if (dtype == QD_F32) GO(float, false); else GO(bf16, false); }
#undef GO
#undef GO2
  return qd_last_error();
}

// ------------------------------------------------------------------------------ the residual sum's norm
#define NORM_MAX_BLOCKS (32 * 16)             // 65,536 features
struct NormArgs {
  float* x;
  const void* delta;
  const float *dscale, *w;
  unsigned char *q, *s;
  const int* rows;
  int D, blocks, n_parts, write_back;
  float eps;
  long long part_stride, ldq, lds;
};

// One CTA to a row.  A warp holds up to VPT of the row's blocks in registers.  The squares are summed block by block, a block in the order of
// a warp's butterfly, the blocks' sums by lanes and then such a butterfly: an order that depends only on D, whatever VPT the number of rows
// leads to, so that a row's result does not depend on what else is in the batch.
template <typename TD, int VPT, bool VEC>
__global__ void __launch_bounds__(1024) norm_fp8_kernel(const NormArgs a) {
  __shared__ float squares[32 * VPT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, step = (blockDim.x >> 5) * FP8_BLOCK, k0 = warp * FP8_BLOCK + 4 * lane;
  pdl_launch_dependents();
  pdl_wait();
  // (after the wait, as all that is read: the launch before may have written the weights; with few blocks to a warp they travel beside the row)
  float4 w[VPT <= 4 ? VPT : 1];
  if (VPT <= 4)
#pragma unroll
    for (int i = 0; i < VPT; i++) w[VPT <= 4 ? i : 0] = load4<VEC>(a.w, k0 + i * step, a.D);
  const int r = blockIdx.x;
  const size_t at = (size_t)(a.rows ? a.rows[r] : r) * a.D;
  float4 v[VPT];
#pragma unroll
  for (int i = 0; i < VPT; i++) v[i] = load4<VEC>(a.x + at, k0 + i * step, a.D);
  if (a.delta) {
    float4 d[VPT];
    sum_parts<VEC>(d, (const TD*)a.delta + at, k0, step, a.D, a.n_parts, a.part_stride);
#pragma unroll
    for (int i = 0; i < VPT; i++) {
      const int k = k0 + i * step;
      if (a.dscale) {
        const float4 f = load4<VEC>(a.dscale, k, a.D);
        v[i].x = fmaf(d[i].x, f.x, v[i].x); v[i].y = fmaf(d[i].y, f.y, v[i].y); v[i].z = fmaf(d[i].z, f.z, v[i].z); v[i].w = fmaf(d[i].w, f.w, v[i].w);
      } else {
        add4(v[i], d[i]);
      }
      if (a.write_back) {
        float* to = a.x + at + k;
        if (VEC) {
          if (k < a.D) *reinterpret_cast<float4*>(to) = v[i];
        } else {
          if (k < a.D) to[0] = v[i].x;
          if (k + 1 < a.D) to[1] = v[i].y;
          if (k + 2 < a.D) to[2] = v[i].z;
          if (k + 3 < a.D) to[3] = v[i].w;
        }
      }
    }
  }
  // The butterflies of VPT blocks as one: of two sums a lane keeps one, and gives the other to the lane that keeps that
  float sq[VPT];
#pragma unroll
  for (int i = 0; i < VPT; i++) sq[i] = fmaf(v[i].w, v[i].w, fmaf(v[i].z, v[i].z, fmaf(v[i].y, v[i].y, v[i].x * v[i].x)));
#pragma unroll
  for (int o = 16, n = VPT / 2; o; o >>= 1, n >>= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < (n ? n : 1); i++) {
      const float next = sq[(i + n) % VPT], other = n && !upper ? next : sq[i];
      if (n && upper) sq[i] = next;
      sq[i] += __shfl_xor_sync(0xffffffffu, other, o);
    }
  }
  const int of = warp + lane / (32 / VPT) * (int)(blockDim.x >> 5);
  if (lane % (32 / VPT) == 0 && of < a.blocks) squares[of] = sq[0];
  __syncthreads();
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; i++) ss += lane + 32 * i < a.blocks ? squares[lane + 32 * i] : 0.f;
  ss = warp_sum(ss);
  const float inv = 1.0f / sqrtf(ss / (float)a.D + a.eps);
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const int block = warp + i * (int)(blockDim.x >> 5);
    if (block < a.blocks) {
      const float4 f = VPT <= 4 ? w[VPT <= 4 ? i : 0] : load4<VEC>(a.w, k0 + i * step, a.D);
      v[i].x = v[i].x * inv * f.x; v[i].y = v[i].y * inv * f.y; v[i].z = v[i].z * inv * f.z; v[i].w = v[i].w * inv * f.w;
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
  const bool vec = D % 4 == 0 && part_stride % 4 == 0 && !(((uintptr_t)x | (uintptr_t)w | (uintptr_t)dscale) & 15) &&
          !((uintptr_t)delta & (delta_dtype == QD_BF16 ? 7 : 15));
  if (a.blocks > NORM_MAX_BLOCKS) return QD_ERR_UNSUPPORTED;
  // As many rows as run at a time (64 warps to a multiprocessor): a block to each warp, the shortest way; more: four, so that more rows are
  // on their way at a time (512 and 2,048 rows of 2,048 features, us: 3.3 and 11.0 with one, 4.6 and 9.8 with four)
  const int vpt = a.blocks > 128 ? 16 : a.blocks > 64 ? 4 : a.blocks > 32 ? (n_rows > 296 ? 4 : 2) : n_rows > 148 * (64 / a.blocks) ? 4 : 1;
  const dim3 grid(n_rows), block(32 * ((a.blocks + vpt - 1) / vpt));
#define GO(TD, V) do { if (vec) qd_launch(norm_fp8_kernel<TD, V, true>, grid, block, 0, stream, a);                           \
                       else qd_launch(norm_fp8_kernel<TD, V, false>, grid, block, 0, stream, a); } while (0)
#define PICK(TD) do { if (vpt == 1) GO(TD, 1); else if (vpt == 2) GO(TD, 2); else if (vpt == 4) GO(TD, 4); else GO(TD, 16); } while (0)
  if (delta && delta_dtype == QD_BF16) PICK(bf16); else PICK(float);
#undef PICK
#undef GO
  return qd_last_error();
}
