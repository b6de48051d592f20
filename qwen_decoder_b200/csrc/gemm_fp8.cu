// Contraction Y[T, N] = X[T, K] * W[N, K]^T of rows in 8 bits (fp8.cuh) on the tensor cores, which apply the scales themselves:
//
//   Y[t, n] = sum_b 2^(ex[t, b] + ew[n, b]) sum_{k in block b} x[t, k] w[n, k]
//
// tcgen05.mma kind::mxf8f6f4 with block scaling takes e4m3 operands from shared memory (TMA tensor copies, 128-byte swizzle, a block of
// 128 k to a stage), float32 sums in tensor memory and the scales, bytes of exponents, from tensor memory too: lane l, column c of a
// tile's scales holds the scales of row 32 c + l, the same in all four quarters of the lanes.  A column's word has four bytes and the
// instruction says which one it takes, so a word is the scales of four blocks of 128 k: exactly four neighbouring bytes of a row of
// scales.  Four warps of a CTA bring these words, one for each quarter.
//
// One CTA to a tile of up to 128 tokens, or (``CG`` 2) two to a tile of up to 256: each brings its own tokens and half of the weights'
// rows, the tensor cores of both read both halves.  A worker (a CTA or a pair) goes through its items one after the other with two
// accumulators in turn, so that an item's epilogue runs under the next one's MMAs.  512 columns of tensor memory hold four buffers of
// scales (64 columns) and two accumulators of up to 224 columns; two of 256 overlap in 64 columns, which the epilogue reads first, and
// then lets the next item's MMAs begin.
//
// Warps: 0..7 epilogue (two for each quarter of the lanes, columns halved between them), 8 producer, 9 MMAs, 10..13 scales.
//
// Epilogues: whole sums (+ bias) as bfloat16 or float32; the same of a K shared by the CTAs of a cluster, joined over their shared
// memories in the order of the shares; the gated activation in 8 bits, where a tile has 128 features of the gate matrix and the same of
// the up matrix, a block of the result's rows, whose largest magnitude the two warps of a row exchange.
//
// Every mbarrier wait is bounded; after one that ran out all roles run on to their ends with void results and a status word says
// which wait it was.
//
// The reference has 16-bit products only (cublasHgemm, gpu_kernels.cu:431-436).
#include "entry_points.h"
#include "fp8.cuh"
#include "tc5_ops.cuh"

#define G8_EPI_WARPS 8
#define G8_THREADS (14 * 32)
#define G8_MAX_STAGES 16
#define G8_SMEM (202 * 1024)                  // of stages
#define G8_WORDS 4                            // of scales that are brought together
#define G8_STAGE_ROWS (32 * 64)               // of a warp's epilogue: 64 bytes of each of its rows
#define G8_MAX_SMEM (G8_SMEM + G8_EPI_WARPS * G8_STAGE_ROWS + 1024)
#define G8_COLS 512                           // of tensor memory, all
#define G8_SCALES 448                         // columns of the scales' buffers, 16 each: 4 of the tokens', up to 8 of the weights'
#define G8_BUFFERS 4
#define G8_FEW 16                             // tokens of a gated product whose sums fit the epilogue's part of shared memory
#define G8_OVERLAP 64                         // columns that two accumulators of 256 share (the first that the epilogue reads)

#define G8_STORE QD_FP8_STORE
#define G8_SHARED 1                           // K shared by a cluster
#define G8_GATED QD_FP8_GATED

struct G8Params {
  int act, T, N, K;
  int bn;                  // rows of W of a tile, of both CTAs together
  int mrows;               // tokens of a CTA
  int n_ft, n_tt, splits;
  int kb_total, stages;
  int feats;               // columns of the result
  int vec;                 // rows of the result take 16-byte stores
  int resident;            // no kernel before this one writes W or its scales
  long long ldo;           // elements
  const unsigned char *sx, *sw;
  long long ldsx, ldsw;
  int doubt;               // of the gated product, as what follows
  const unsigned char *x, *w;
  long long ldx, ldw;
  unsigned char* s_out;
  long long lds_out;
};

// ---- what a pair needs beyond tc5_ops.cuh
__device__ __forceinline__ unsigned g8_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
// where the first CTA of the pair has what this one has at ``p``: bit 24 of a shared-memory address is the place in the pair
__device__ __forceinline__ unsigned g8_leader(const void* p) { return tc_smem(p) & 0xFEFFFFFFu; }
__device__ __forceinline__ void g8_arrive_at(unsigned bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void g8_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void g8_load_2d(void* dst, const CUtensorMap* map, int x, int y, unsigned bar) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(tc_smem(dst)), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
template <int CG>
__device__ __forceinline__ void g8_mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned sa, unsigned sb,
                                       bool accumulate) {
  if (CG == 2)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate ? 1u : 0u) : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate ? 1u : 0u) : "memory");
}
// e4m3 operands, both K-major, scales of 8 exponent bits; the scales' byte is added for each MMA
__device__ __forceinline__ unsigned g8_idesc(int m, int n) { return (unsigned)(n >> 3) << 17 | 1u << 23 | (unsigned)(m >> 4) << 24; }
__device__ __forceinline__ unsigned g8_idesc_byte(unsigned i) { return i << 4 | i << 29; }
// arrives at the barrier of both CTAs once the MMAs so far are done
template <int CG>
__device__ __forceinline__ void g8_commit(unsigned long long* bar) {
  if (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(tc_smem(bar)), "h"((unsigned short)3) : "memory");
  else tc_commit(bar);
}
__device__ __forceinline__ void g8_ld16(unsigned addr, float (&v)[16]) {
  unsigned r[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr));
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void g8_st4(unsigned addr, const unsigned* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}

// a row's scales of the next four blocks of 128 k, or the ``there`` that there are
__device__ __forceinline__ unsigned g8_scales(const unsigned char* s, int there) {
  if (there >= 4) return *reinterpret_cast<const unsigned*>(s);
  unsigned v = s[0];
  if (there > 1) v |= s[1] << 8;
  if (there > 2) v |= s[2] << 16;
  return v;
}

// A worker's item
struct G8Item { int tt, ft, kb0, kb1; };
__device__ __forceinline__ G8Item g8_item(const G8Params& p, int item, int share) {
  G8Item q;
  q.tt = item % p.n_tt;
  q.ft = item / p.n_tt;
  q.kb0 = p.kb_total * share / p.splits;
  q.kb1 = p.kb_total * (share + 1) / p.splits;
  return q;
}

// The tensor cores cut a sum off at 24 bits with every addition, always towards zero: 4 additions to a block of 128 k, 2.7e-7 of the sum's
// norm after 512 of k, 1.7e-6 after 3,584 (scales spread over 2^12).  A float32 result is therefore summed in pieces of 1,024 of k, which
// the epilogue adds up with rounding (5e-7); what becomes bfloat16 is off by 1.7e-3 anyway and stays one sum.
#define G8_PIECE 8
#define G8_MAX_FLOAT_BN 128                   // of which a thread of the epilogue keeps half a row's sums
template <typename TO>
__device__ __forceinline__ int g8_piece_end(const G8Item& q, int kb) { return sizeof(TO) == 4 ? min(kb + G8_PIECE, q.kb1) : q.kb1; }

__device__ __forceinline__ void g8_bias16(float (&v)[16], const float* bias, int col, int feats) {
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (col + i < feats) v[i] += bias[col + i];
}
// 16 numbers as pieces of 16 bytes of a row of 64 in a warp's part of shared memory.  Rows lie side by side, the pieces of rows
// 2 i and 2 i + 1 turned by i: eight lanes that write or read together meet no bank twice.
__device__ __forceinline__ uint4* g8_piece(unsigned char* rows, int row, int piece) {
  return reinterpret_cast<uint4*>(rows + row * 64 + ((piece ^ (row >> 1 & 3)) << 4));
}
__device__ __forceinline__ unsigned g8_bf16x2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <typename TO>
__device__ __forceinline__ void g8_stage16(unsigned char* rows, int row, int piece, const float (&v)[16]) {
  if (sizeof(TO) == 4) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      *g8_piece(rows, row, piece + i) = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                                                   __float_as_uint(v[4 * i + 3]));
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++)
      *g8_piece(rows, row, piece + i) = make_uint4(g8_bf16x2(v[8 * i], v[8 * i + 1]), g8_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                                                   g8_bf16x2(v[8 * i + 4], v[8 * i + 5]), g8_bf16x2(v[8 * i + 6], v[8 * i + 7]));
  }
}
// The first ``pieces`` of the four pieces of each of a warp's first ``n_rows`` rows to memory, ``left`` elements of a row from ``dst`` on
template <typename TO>
__device__ __forceinline__ void g8_store_rows(unsigned char* rows, TO* dst, long long ld, int n_rows, int pieces, int left, bool vec) {
  constexpr int E = 16 / (int)sizeof(TO);
  const int lane = threadIdx.x & 31;
  if (vec && left >= pieces * E) {
    const int piece = lane & 3;
    if (piece >= pieces) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = 8 * i + (lane >> 2);
      if (r < n_rows) *reinterpret_cast<uint4*>(dst + (size_t)r * ld + piece * E) = *g8_piece(rows, r, piece);
    }
  } else {
    // a row at a time, its elements side by side
    const int n = min(left, pieces * E);
    for (int r = 0; r < n_rows; r++)
      for (int e = lane; e < n; e += 32) dst[(size_t)r * ld + e] = reinterpret_cast<const TO*>(g8_piece(rows, r, e / E))[e % E];
  }
}

// h = act(g) u of 64 features from ``col0`` on, zero from ``feats`` on: h holds the gate's sums (``gate``) or up's, the others lie in tensor
// memory
template <int ACT>
__device__ __forceinline__ void g8_activate(float (&h)[64], unsigned other, bool gate, const float* bias, int col0, int feats, float& deepest) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float o[16];
    float (&x)[16] = *reinterpret_cast<float (*)[16]>(h + 16 * i);
    g8_ld16(other + 16 * i, o);
    tc_ld_wait();
    if (bias) {
      g8_bias16(x, bias + (gate ? 0 : feats), col0 + 16 * i, feats);
      g8_bias16(o, bias + (gate ? feats : 0), col0 + 16 * i, feats);
    }
#pragma unroll
    for (int e = 0; e < 16; e++) {
      deepest = fminf(deepest, gate ? x[e] : o[e]);
      x[e] = fp8_gated_short(gate ? x[e] : o[e], gate ? o[e] : x[e], ACT);
    }
    if (col0 + 16 * i + 16 > feats)
#pragma unroll
      for (int e = 0; e < 16; e++)
        if (col0 + 16 * i + e >= feats) x[e] = 0.f;
  }
}

// Where a block's largest magnitude is so near the last one of a scale that the sums' cut-off decides, its sums are made again at the kernel's
// end: a scale is then that of the sums as they are, not of the order of their additions.  (Without it 1 to 4 of a million blocks had the
// other scale, K 2,048 to 11,008; some 25 of a million are looked at for K 3,584, 2 to 3 us each where the kernel ends with one: a layer of 8
// tokens of the 7B sizes 56.6 -> 57.3 us.  Looked at in the epilogue itself they made its code so long that products of 8 to 512 tokens took 3
// to 15 % more.)  How near is in units of the last place at 1.75: K / 32 additions, cut off by 0.02 to 0.09 of a unit each, by up to 0.2
// in most sums of numbers of one sign, in the gate's sum and in up's, and the activation's own error (1.75 times 5, and what the deepest gate
// adds), which the look itself does not have: where it counts it goes on in float64 to the end.  Each thread tells of its own features, so that
// a block may come twice; the second look finds it as it has to be.  (A gate of -g < -2 makes g - 1 times its sum's error of it: where every
// gate of a block lies far below -10, sums of one sign may leave the other scale, which holds the block as well but for half a step.)
// blocks that a CTA keeps for that; with more of them it goes through all that it has written, a tile's at a time
#define G8_NEAR 128
static int g8_doubt(int K) { return K < 1 << 24 ? (K >> 5) + 16 : 0xfffff; }
#define G8_448 0x7e                           // as e4m3
#define G8_224 0x76
// ``most``: the largest magnitude of a block; ``peak``: that of some of its features, the lowest of whose gates is ``deepest`` (0, or below).  (Where
// the activation is zero it has no error.)
__device__ __forceinline__ bool g8_near(unsigned most, float peak, float deepest, int doubt, int act) {
  const bool gelu = act == QD_ACT_GELU_TANH;
  const int off = (int)(most & 0x7fffffu) - 0x600000;
  if (most < 10u << 23 || most >= 0x7f800000u || abs(off) > doubt + (gelu ? 570 : 185)) return false;
  const int margin = doubt - (int)(qd_gate_arg(fmaxf(deepest, gelu ? -10.f : -88.f), act) * (gelu ? 6.5f : 2.1f));
  return abs((int)__float_as_uint(peak) - (int)most + off) <= margin;
}
// 8 e4m3 numbers of a row, zeros behind its end
__device__ __forceinline__ void g8_eight(float (&v)[8], const unsigned char* from, int there) {
  uint2 raw = make_uint2(0, 0);
  if (there >= 8) {
    raw = *reinterpret_cast<const uint2*>(from);
  } else {
#pragma unroll 1
    for (int i = 0; i < there; i++) (i < 4 ? raw.x : raw.y) |= (unsigned)from[i] << 8 * (i & 3);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    unsigned h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)((i < 2 ? raw.x : raw.y) >> 16 * (i & 1))));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
// 2^(a + b) of two scales' bytes
__device__ __forceinline__ double g8_scaled(unsigned a, unsigned b) { return __longlong_as_double((long long)(a + b - 254 + 1023) << 52); }

template <int ACT>
struct G8Act { static constexpr int value = ACT; };

template <int EPI, typename TO, int CG>
__global__ void __launch_bounds__(G8_THREADS, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const float* bias,
                TO* __restrict__ out, const G8Params p, int* __restrict__ status) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ unsigned long long full[G8_MAX_STAGES], empty[G8_MAX_STAGES], acc_ready[2], acc_free[2], scales_full[G8_BUFFERS], scales_empty[G8_BUFFERS];
  __shared__ unsigned tmem_slot, peaks[4][2][32], scales[G8_WORDS][384];
  __shared__ int dead, n_near;
  __shared__ unsigned near_rows[EPI == G8_GATED ? G8_NEAR : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? (int)g8_rank() : 0;
  const int share = EPI == G8_SHARED ? (int)g8_rank() : 0;
  unsigned char* base = smem_raw + ((1024 - (tc_smem(smem_raw) & 1023)) & 1023);
  // The stages' tokens lie before the stages' weights: an MMA reads 128 rows of tokens whatever a CTA has, and what lies behind
  // them is then always there.
  const int a_bytes = p.mrows * 128, b_bytes = p.bn / CG * 128;
  unsigned char* a_s = base;
  unsigned char* b_s = base + (size_t)p.stages * a_bytes;
  if (threadIdx.x == 0) {
    dead = n_near = 0;
    for (int s = 0; s < p.stages; s++) { tc_bar_init(&full[s], 1); tc_bar_init(&empty[s], 1); }
    for (int b = 0; b < 2; b++) {
      tc_bar_init(&acc_ready[b], 1);
      tc_bar_init(&acc_free[b], CG * G8_EPI_WARPS);
    }
    for (int b = 0; b < G8_BUFFERS; b++) { tc_bar_init(&scales_full[b], CG == 2 && rank == 0 ? 5 : 4); tc_bar_init(&scales_empty[b], 1); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (CG == 2) g8_cluster_sync();

  const int per = EPI == G8_SHARED ? p.splits : CG;
  const int worker = blockIdx.x / per, n_workers = gridDim.x / per, n_items = p.n_ft * p.n_tt;
  const int half = p.bn >> 1;
  const bool overlap = p.bn > G8_SCALES / 2;
  const unsigned acc_step = overlap ? 256 - G8_OVERLAP : G8_SCALES / 2;
  auto row_x = [&](const G8Item& q) { return (CG * q.tt + rank) * p.mrows; };
  // the first row of W of the part ``h`` (0: first half, 1: second) of an item's tile
  auto row_w = [&](const G8Item& q, int h) { return EPI == G8_GATED ? q.ft * half + h * p.feats : q.ft * p.bn + h * half; };

  if (warp == G8_EPI_WARPS) {
    // ------------------------------------------------------------------ producer
    // (the whole warp goes through the loop and one lane issues: addresses and coordinates are then known to be the same for all lanes)
    const bool one = tc_elect();
    const unsigned bytes = (unsigned)(CG * (a_bytes + b_bytes));
    auto load = [&](unsigned char* dst, const CUtensorMap* map, int x, int y, int s) {
      if (CG == 2) g8_load_2d(dst, map, x, y, g8_leader(&full[s]));
      else tc_load_2d(dst, map, x, y, &full[s]);
    };
    auto tokens = [&](int s, const G8Item& q, int kb) { load(a_s + s * a_bytes, &map_x, kb * FP8_BLOCK, row_x(q), s); };
    auto weights = [&](int s, const G8Item& q, int kb) {
      if (CG == 1 || rank == 0) tc_expect_tx(&full[s], bytes);
      load(b_s + s * b_bytes, &map_w, kb * FP8_BLOCK, row_w(q, rank), s);
      if (CG == 1 && EPI == G8_GATED) load(b_s + s * b_bytes + half * 128, &map_w, kb * FP8_BLOCK, row_w(q, 1), s);
    };
    int item = worker, n = 0;
    G8Item q = g8_item(p, item, share);
    int kb = q.kb0;
    auto next = [&](int& it, G8Item& i, int& k) {
      if (++k < i.kb1) return;
      it += n_workers;
      if (it < n_items) i = g8_item(p, it, share);
      k = i.kb0;
    };
    int item_t = item, kb_t = kb;
    G8Item q_t = q;
    if (!p.resident) pdl_wait();
    for (; n < p.stages && item < n_items; n++, next(item, q, kb))
      if (one) weights(n, q, kb);
    pdl_wait();
    for (int s = 0; s < n; s++, next(item_t, q_t, kb_t))
      if (one) tokens(s, q_t, kb_t);
    int s = n == p.stages ? 0 : n;
    unsigned ph = 0;
    for (; item < n_items; next(item, q, kb)) {
      if (!tc_wait(&empty[s], ph, &dead)) atomicExch(status, 1);
      if (one) {
        weights(s, q, kb);
        tokens(s, q, kb);
      }
      if (++s == p.stages) { s = 0; ph ^= 1; }
    }
    // the commits' last arrivals at this CTA's barriers come before it may go
    for (int i = 0; i < n; i++) {
      if (n == p.stages) {
        if (!tc_wait(&empty[s], ph, &dead)) atomicExch(status, 1);
        if (++s == p.stages) { s = 0; ph ^= 1; }
      } else if (!tc_wait(&empty[i], 0, &dead)) {
        atomicExch(status, 1);
      }
    }
    __syncwarp();
  } else if (warp == G8_EPI_WARPS + 1) {
    // ------------------------------------------------------------------ MMAs
    if (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(&tmem_slot)), "r"((unsigned)G8_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tc_alloc(&tmem_slot, G8_COLS);
    }
    // (not before this CTA has its tensor memory: the next kernel's CTA beside it might take that, and then wait for this one)
    pdl_launch_dependents();
    tc_fence_before();
    asm volatile("bar.sync 1, %0;" ::"n"(G8_THREADS - 32) : "memory");
    tc_fence_after();
    if (rank == 0) {
      const bool one = tc_elect();
      const unsigned tmem = tmem_slot;
      const unsigned idesc = g8_idesc(128 * CG, p.bn);
      const unsigned long long a0 = tc_desc_sw128(tc_smem(a_s)), b0 = tc_desc_sw128(tc_smem(b_s));
      const unsigned a_step = (unsigned)a_bytes >> 4, b_step = (unsigned)b_bytes >> 4;
      int s = 0, n = 0;
      unsigned ph = 0, sc = 0, sc_ph = 0;
      for (int item = worker; item < n_items; item += n_workers) {
        const G8Item q = g8_item(p, item, share);
        for (int k0 = q.kb0; k0 < q.kb1; n++) {
          const int k1 = g8_piece_end<TO>(q, k0);
          const unsigned buf = n & 1;
          // accumulators apart: the sum before the last has been read; overlapping: of the last one the common columns have
          const int of = overlap ? n - 1 : n - 2;
          if (of >= 0 && !tc_wait(&acc_free[of & 1], of >> 1 & 1, &dead)) atomicExch(status, 3);
          tc_fence_after();
          const unsigned d = tmem + buf * acc_step;
          for (int kb = k0; kb < k1; kb++) {
            if ((kb == q.kb0 || !(kb & 3)) && !tc_wait(&scales_full[sc], sc_ph, &dead)) atomicExch(status, 5);
            if (!tc_wait(&full[s], ph, &dead)) atomicExch(status, 2);
            tc_fence_after();
            const unsigned long long da = a0 + s * a_step, db = b0 + s * b_step;
            const unsigned id = idesc | g8_idesc_byte(kb & 3), sa = tmem + G8_SCALES + 16 * sc;
            const bool last = kb + 1 == q.kb1 || (kb & 3) == 3;
            if (one) {
#pragma unroll
              for (int k = 0; k < FP8_BLOCK / 32; k++) g8_mma<CG>(d, da + 2 * k, db + 2 * k, id, sa, sa + 4, k > 0 || kb > k0);
              g8_commit<CG>(&empty[s]);
              if (last) g8_commit<CG>(&scales_empty[sc]);
            }
            if (last && ++sc == G8_BUFFERS) { sc = 0; sc_ph ^= 1; }
            if (++s == p.stages) { s = 0; ph ^= 1; }
          }
          if (one) g8_commit<CG>(&acc_ready[buf]);
          k0 = k1;
        }
      }
    } else {
      // The pair's second CTA: its scales are there, word by word.  An arrival at the first CTA's barrier waits for the loads before it;
      // from the warps that load the scales it was the time of the whole (2,048 x 8,192 x 2,048 in tiles of 256 x 256 35.2 us, x 128 49.5;
      // without the scales' loads 31.1 and 37.3), so this warp, which has none, hands them on.
      int words = 0;
      for (int item = worker; item < n_items; item += n_workers) {
        const G8Item q = g8_item(p, item, share);
        for (int kw = q.kb0 >> 2; kw <= (q.kb1 - 1) >> 2; kw++, words++) {
          const int sc = words % G8_BUFFERS;
          if (!tc_wait(&scales_full[sc], words / G8_BUFFERS & 1, &dead)) atomicExch(status, 5);
          tc_fence_after();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) g8_arrive_at(g8_leader(&scales_full[sc]));
        }
      }
    }
    __syncwarp();
  } else if (warp >= G8_EPI_WARPS + 2) {
    // ------------------------------------------------------------------ scales
    asm volatile("bar.sync 1, %0;" ::"n"(G8_THREADS - 32) : "memory");
    tc_fence_after();
    const unsigned at = tmem_slot + ((unsigned)(warp & 3) << 21) + G8_SCALES;
    const int wcols = (p.bn + 31) >> 5;
    // A thread brings three rows' words, a token's and two of W, G8_WORDS of each together and the next ones while the present ones are
    // handed out; each warp then takes all 384 rows' from shared memory.  (With every warp loading all rows itself, word by word, the
    // loads of rows 148 bytes apart were the time of 2,048 x 3,584 x 18,944 in pairs: 174 us, so 121.)
    const int t = threadIdx.x - (G8_EPI_WARPS + 2) * 32;
    const unsigned char* from[3];
    unsigned v[3][G8_WORDS];
    int item = worker, kw = 0, kw_end = 0, words = 0;
    auto open = [&]() {
      const G8Item q = g8_item(p, item, share);
      kw = q.kb0 >> 2;
      kw_end = ((q.kb1 - 1) >> 2) + 1;
      const int row = row_x(q) + t;
      from[0] = t < p.mrows && row < p.T ? p.sx + row * p.ldsx : nullptr;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int j = t + 128 * i, h = j >= half, row_of_w = row_w(q, h) + j - (h ? half : 0);
        from[1 + i] = j < p.bn && row_of_w < p.N ? p.sw + row_of_w * p.ldsw : nullptr;
      }
    };
    auto load = [&](int i) {
      const int n = min(G8_WORDS, kw_end - kw);
#pragma unroll
      for (int k = 0; k < G8_WORDS; k++) v[i][k] = from[i] && k < n ? g8_scales(from[i] + 4 * (kw + k), p.kb_total - 4 * (kw + k)) : 0;
    };
    auto next = [&]() {                                      // how many words the loads before were of
      const int n = min(G8_WORDS, kw_end - kw);
      kw += n;
      if (kw == kw_end) {
        item += n_workers;
        if (item < n_items) open();
      }
      return n;
    };
    open();
    if (!p.resident) pdl_wait();
    load(1);
    load(2);
    pdl_wait();
    load(0);
    for (int n = next(); n;) {
      asm volatile("bar.sync 6, 128;" ::: "memory");         // the words before have been taken
#pragma unroll
      for (int i = 0; i < 3; i++)
#pragma unroll
        for (int k = 0; k < G8_WORDS; k++) scales[k][t + 128 * i] = v[i][k];
      asm volatile("bar.sync 6, 128;" ::: "memory");
      const int now = n;
      n = 0;
      if (item < n_items) {
#pragma unroll
        for (int i = 0; i < 3; i++) load(i);
        n = next();
      }
      for (int k = 0; k < now; k++, words++) {
        const int sc = words % G8_BUFFERS;
        unsigned w[12];
#pragma unroll
        for (int c = 0; c < 12; c++) w[c] = scales[k][32 * c + lane];
        if (!tc_wait(&scales_empty[sc], ~(words / G8_BUFFERS) & 1, &dead)) atomicExch(status, 6);
        tc_fence_after();
        g8_st4(at + 16 * sc, w);
        g8_st4(at + 16 * sc + 4, w + 4);
        if (wcols > 4) g8_st4(at + 16 * sc + 8, w + 8);
        tc_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) tc_arrive(&scales_full[sc]);
      }
    }
    // the commits' last arrivals at these barriers, too
    for (int i = max(0, words - G8_BUFFERS); i < words; i++)
      if (!tc_wait(&scales_empty[i % G8_BUFFERS], i / G8_BUFFERS & 1, &dead)) atomicExch(status, 6);
  } else {
    // ------------------------------------------------------------------ epilogue
    asm volatile("bar.sync 1, %0;" ::"n"(G8_THREADS - 32) : "memory");
    tc_fence_after();
    const int quarter = (warp & 3) * 32, side = warp >> 2;
    const unsigned tmem = tmem_slot + ((unsigned)quarter << 16);
    unsigned char* rows = b_s + (size_t)p.stages * b_bytes + warp * G8_STAGE_ROWS;
    auto release = [&](unsigned buf) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2) g8_arrive_at(g8_leader(&acc_free[buf]));
        else tc_arrive(&acc_free[buf]);
      }
    };
    // 16 columns of a share of K as float32, a row's pieces turned by the row: what the cluster adds up
    auto keep16 = [&](const float (&v)[16], int g) {
#pragma unroll
      for (int e = 0; e < 4; e++)
        *reinterpret_cast<float4*>(base + (size_t)(quarter + lane) * p.bn * 4 + ((4 * g + e ^ (lane & 7)) << 4)) =
            make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
    };
    // a row of the item's tile whose scale is to be looked at
    auto look_at = [&](int item, int r) {
      const int at = atomicAdd(&n_near, 1);
      if (at < G8_NEAR) near_rows[at] = (unsigned)item << 7 | r;
    };
    int n = 0;
    auto wait_sum = [&]() {
      if (!tc_wait(&acc_ready[n & 1], n >> 1 & 1, &dead, 64) && lane == 0) atomicExch(status, 4);
      tc_fence_after();
    };
    for (int item = worker; item < n_items; item += n_workers) {
      const G8Item q = g8_item(p, item, share);
      const int tok0 = row_x(q) + quarter;                   // of this warp's rows the first, and how many there are
      const int n_rows = min(32, min(p.mrows - quarter, p.T - tok0));
      const int groups = p.bn / 16, g0 = groups * side / 2, g1 = groups * (side + 1) / 2;     // this side's 16s of columns
      if constexpr (sizeof(TO) == 4) {
        constexpr int MOST = G8_MAX_FLOAT_BN / 32;
        float sum[MOST][16];
        for (int k0 = q.kb0; k0 < q.kb1; k0 = g8_piece_end<TO>(q, k0), n++) {
          wait_sum();
          const unsigned acc = tmem + (n & 1) * acc_step;
          if (n_rows > 0) {                                  // whole warps: the loads are collective
#pragma unroll
            for (int i = 0; i < MOST; i++)
              if (i < g1 - g0) {
                float v[16];
                g8_ld16(acc + 16 * (g0 + i), v);
                tc_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; e++) sum[i][e] = k0 == q.kb0 ? v[e] : sum[i][e] + v[e];
              }
          }
          release(n & 1);
        }
        if (n_rows > 0) {
#pragma unroll
          for (int i = 0; i < MOST; i++)
            if (i < g1 - g0) {
              const int col = q.ft * p.bn + 16 * (g0 + i);
              if constexpr (EPI == G8_SHARED) {
                if (lane < n_rows) keep16(sum[i], g0 + i);
              } else {
                if (bias) g8_bias16(sum[i], bias, col, p.feats);
                __syncwarp();
                g8_stage16<TO>(rows, lane, 0, sum[i]);
                __syncwarp();
                g8_store_rows<TO>(rows, out + (size_t)tok0 * p.ldo + col, p.ldo, n_rows, 4, p.feats - col, p.vec);
              }
            }
        }
        continue;
      }
      const unsigned buf = n & 1;
      wait_sum();
      n++;
      const unsigned acc = tmem + buf * acc_step;
      // which side has the columns that overlap with the next item's: the first accumulator's last, the second's first
      const bool owner = overlap && side == (buf == 0);
      if (overlap && (!owner || n_rows <= 0)) release(buf);
      if constexpr (EPI == G8_GATED) {
        const bool only = CG == 1 && n_items <= n_workers;   // (its stages have all been read)
        if (p.mrows <= G8_FEW || (only && p.mrows <= 32)) {
          // The rows of few tokens lie in one quarter of the lanes, which two of the warps reach: they pass the sums on through shared
          // memory, a row of 256 to a warp, four features to a lane (two warps alone took 16.3 us for 8 tokens of 2,048 by 2 x 11,008).
          float* sums = reinterpret_cast<float*>(only ? base : b_s + (size_t)p.stages * b_bytes);
          if (quarter == 0) {
#pragma unroll 1
            for (int i = 0; i < 8; i++) {
              const int g = owner && side ? 15 - i : 8 * side + i;
              float v[16];
              g8_ld16(acc + 16 * g, v);
              tc_ld_wait();
              if (owner && n_rows > 0 && i == G8_OVERLAP / 16 - 1) release(buf);       // (a CTA without rows has done so above)
              if (lane < n_rows)
#pragma unroll
                for (int e = 0; e < 4; e++)
                  *reinterpret_cast<float4*>(sums + lane * 256 + ((4 * g + e ^ (lane & 7)) << 2)) =
                      make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
            }
          }
          asm volatile("bar.sync 7, 256;" ::: "memory");
          const int tokens = min(p.mrows, p.T - row_x(q)), col = q.ft * 128 + 4 * lane;
          const auto gate = [&](auto act) {
#pragma unroll 1
            for (int r = warp; r < tokens; r += G8_EPI_WARPS) {
              const float4 g4 = *reinterpret_cast<const float4*>(sums + r * 256 + ((lane ^ (r & 7)) << 2));
              const float4 u4 = *reinterpret_cast<const float4*>(sums + r * 256 + ((32 + lane ^ (r & 7)) << 2));
              float g[4] = {g4.x, g4.y, g4.z, g4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w};
              float peak = 0.f, deepest = 0.f;
#pragma unroll
              for (int e = 0; e < 4; e++) {
                if (bias && col + e < p.feats) {
                  g[e] += bias[col + e];
                  u[e] += bias[p.feats + col + e];
                }
                deepest = fminf(deepest, g[e]);
                g[e] = fp8_gated_short(g[e], u[e], decltype(act)::value);
              }
              if (col + 4 > p.feats)
#pragma unroll
                for (int e = 0; e < 4; e++)
                  if (col + e >= p.feats) g[e] = 0.f;
#pragma unroll
              for (int e = 0; e < 4; e++) peak = fp8_peak(peak, g[e]);
              const unsigned most = __reduce_max_sync(0xffffffffu, __float_as_uint(peak)), byte = fp8_scale_byte(most);
              if (g8_near(most, peak, deepest, p.doubt, decltype(act)::value)) look_at(item, r);
              const float inv = fp8_inverse(byte);
              const unsigned w = fp8_pack4(g[0] * inv, g[1] * inv, g[2] * inv, g[3] * inv);
              unsigned char* to = (unsigned char*)out + (size_t)(row_x(q) + r) * p.ldo + col;
              if (col + 4 <= p.feats) *reinterpret_cast<unsigned*>(to) = w;
              else
                for (int e = 0; e < 4 && col + e < p.feats; e++) to[e] = (unsigned char)(w >> 8 * e);
              if (lane == 0) p.s_out[(size_t)(row_x(q) + r) * p.lds_out + q.ft] = (unsigned char)byte;
            }
          };
          if (p.act == QD_ACT_GELU_TANH) gate(G8Act<QD_ACT_GELU_TANH>());
          else gate(G8Act<QD_ACT_SILU>());
          asm volatile("bar.sync 7, 256;" ::: "memory");     // the sums have been read
        } else if (only) {
          // 16 features at a time, the activations by way of shared memory: the code below, which keeps 64 in registers, is long, and after
          // other launches the wait for it hides behind nothing here (64 tokens, 2,048 by 2 x 11,008 between the launches of a layer: 18.4 us,
          // so 13.6; alone, over and over, 13.3 and 13.1; with the second look at scales 14.8 and 13.5).
          if (n_rows > 0) {
            float4* mine = reinterpret_cast<float4*>(base) + threadIdx.x;
            const int col0 = q.ft * 128 + 64 * side;
            float peak = 0.f, deepest = 0.f;
            const auto gate = [&](auto act) {
#pragma unroll 1
              for (int i = 0; i < 4; i++) {
                float g[16], u[16];
                g8_ld16(acc + 64 * side + 16 * i, g);
                g8_ld16(acc + 128 + 64 * side + 16 * i, u);
                tc_ld_wait();
                const int col = col0 + 16 * i;
                if (bias) {
                  g8_bias16(g, bias, col, p.feats);
                  g8_bias16(u, bias + p.feats, col, p.feats);
                }
#pragma unroll
                for (int e = 0; e < 16; e++) {
                  deepest = fminf(deepest, g[e]);
                  g[e] = fp8_gated_short(g[e], u[e], decltype(act)::value);
                }
                if (col + 16 > p.feats)                      // (asked for each feature by itself: 2.5 us more)
#pragma unroll
                  for (int e = 0; e < 16; e++)
                    if (col + e >= p.feats) g[e] = 0.f;
#pragma unroll
                for (int e = 0; e < 16; e++) peak = fp8_peak(peak, g[e]);
#pragma unroll
                for (int e = 0; e < 4; e++) mine[(4 * i + e) * 32 * G8_EPI_WARPS] = make_float4(g[4 * e], g[4 * e + 1], g[4 * e + 2], g[4 * e + 3]);
              }
            };
            if (p.act == QD_ACT_GELU_TANH) gate(G8Act<QD_ACT_GELU_TANH>());
            else gate(G8Act<QD_ACT_SILU>());
            peaks[warp & 3][side][lane] = __float_as_uint(peak);
            asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory");
            const unsigned most = max(__float_as_uint(peak), peaks[warp & 3][side ^ 1][lane]), byte = fp8_scale_byte(most);
            if (lane < n_rows && g8_near(most, peak, deepest, p.doubt, p.act)) look_at(item, quarter + lane);
            const float inv = fp8_inverse(byte);
#pragma unroll 1
            for (int c = 0; c < 4; c++) {
              unsigned w[4];
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const float4 h = mine[(4 * c + e) * 32 * G8_EPI_WARPS];
                w[e] = fp8_pack4(h.x * inv, h.y * inv, h.z * inv, h.w * inv);
              }
              *g8_piece(rows, lane, c) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
            g8_store_rows<unsigned char>(rows, (unsigned char*)out + (size_t)tok0 * p.ldo + col0, p.ldo, n_rows, 4, p.feats - col0, p.vec);
            if (side == 0 && lane < n_rows) p.s_out[(size_t)(tok0 + lane) * p.lds_out + q.ft] = (unsigned char)byte;
          }
        } else if (n_rows > 0) {                             // whole warps: the loads are collective
          // First the 64 columns that the next item's MMAs may overwrite, of up in the first accumulator and of the gate in the second,
          // then they may begin (with the loads in the activations' order they waited for those: 2,048 tokens of 2,048 by 2 x 11,008
          // 114 us, 1,620 TFLOP/s).
          float h[64], peak = 0.f, deepest = 0.f;
          const unsigned one = acc + 64 * side + (buf ? 0 : 128), two = acc + 64 * side + (buf ? 128 : 0);
#pragma unroll
          for (int i = 0; i < 4; i++) g8_ld16(one + 16 * i, *reinterpret_cast<float (*)[16]>(h + 16 * i));
          tc_ld_wait();
          if (owner) release(buf);
          const int col0 = q.ft * 128 + 64 * side;
          if (p.act == QD_ACT_GELU_TANH) g8_activate<QD_ACT_GELU_TANH>(h, two, buf, bias, col0, p.feats, deepest);
          else g8_activate<QD_ACT_SILU>(h, two, buf, bias, col0, p.feats, deepest);
#pragma unroll
          for (int e = 0; e < 64; e++) peak = fp8_peak(peak, h[e]);
          peaks[warp & 3][side][lane] = __float_as_uint(peak);
          asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory");
          const unsigned most = max(__float_as_uint(peak), peaks[warp & 3][side ^ 1][lane]), byte = fp8_scale_byte(most);
          if (lane < n_rows && g8_near(most, peak, deepest, p.doubt, p.act)) look_at(item, quarter + lane);
          const float inv = fp8_inverse(byte);
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 4; c++) {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
              w[i] = fp8_pack4(h[16 * c + 4 * i] * inv, h[16 * c + 4 * i + 1] * inv, h[16 * c + 4 * i + 2] * inv, h[16 * c + 4 * i + 3] * inv);
            *g8_piece(rows, lane, c) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
          const int col = q.ft * 128 + 64 * side;
          g8_store_rows<unsigned char>(rows, (unsigned char*)out + (size_t)tok0 * p.ldo + col, p.ldo, n_rows, 4, p.feats - col, p.vec);
          if (side == 0 && lane < n_rows) p.s_out[(size_t)(tok0 + lane) * p.lds_out + q.ft] = (unsigned char)byte;
          asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory");        // the peaks have been read
        }
      } else if (n_rows > 0) {
        const int passes = (g1 - g0 + 1) / 2;
        for (int i = 0; i < passes; i++) {
          const int g = owner && side ? g1 - 2 * (i + 1) : g0 + 2 * i;
          const int w = min(2, g1 - g);                      // 64 bytes of every row, or what is left of the columns
          float v[2][16];
#pragma unroll
          for (int j = 0; j < 2; j++)
            if (j < w) g8_ld16(acc + 16 * (g + j), v[j]);
          tc_ld_wait();
          if (owner && i == G8_OVERLAP / 32 - 1) release(buf);
          __syncwarp();
          const int col = q.ft * p.bn + 16 * g;
          if constexpr (EPI == G8_SHARED) {
#pragma unroll
            for (int j = 0; j < 2; j++)
              if (j < w && lane < n_rows) keep16(v[j], g + j);
          } else {
#pragma unroll
            for (int j = 0; j < 2; j++)
              if (j < w) {
                if (bias) g8_bias16(v[j], bias, col + 16 * j, p.feats);
                g8_stage16<TO>(rows, lane, 2 * j, v[j]);
              }
            __syncwarp();
            g8_store_rows<TO>(rows, out + (size_t)tok0 * p.ldo + col, p.ldo, n_rows, 2 * w, p.feats - col, p.vec);
          }
        }
      }
      if (!overlap) release(buf);
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (EPI == G8_SHARED) {
    g8_cluster_sync();
    // this CTA's share of the tile's rows, summed in the order of the shares of K: up to 32 pieces of four features of a row to a warp, two
    // times that on their way together
    const G8Item q = g8_item(p, worker, share);
    const int tok0 = q.tt * p.mrows, n_rows = min(p.mrows, p.T - tok0), pieces = p.bn >> 2, wide = pieces > 32;
    const int r0 = n_rows * share / p.splits, units = (n_rows * (share + 1) / p.splits - r0) << wide;
    const unsigned at = tc_smem(base);
    constexpr int WARPS = G8_THREADS / 32;
#pragma unroll 1
    for (int u0 = warp; u0 < units; u0 += 2 * WARPS) {
      float4 v[2][8];
      int r[2], c[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int u = u0 + h * WARPS;
        r[h] = r0 + (u >> wide);
        c[h] = u < units ? (wide ? (u & 1) * 32 : 0) + lane : pieces;
        const unsigned from = at + (r[h] * pieces + (c[h] ^ (r[h] & 7))) * 16;
#pragma unroll
        for (int sp = 0; sp < 8; sp++)
          if (sp < p.splits && c[h] < pieces) {
            unsigned remote;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(from), "r"(sp));
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v[h][sp].x), "=f"(v[h][sp].y), "=f"(v[h][sp].z), "=f"(v[h][sp].w) : "r"(remote) : "memory");
          }
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if (c[h] >= pieces) break;
        float4 t = v[h][0];
#pragma unroll
        for (int sp = 1; sp < 8; sp++)
          if (sp < p.splits) { t.x += v[h][sp].x; t.y += v[h][sp].y; t.z += v[h][sp].z; t.w += v[h][sp].w; }
        const int col = q.ft * p.bn + 4 * c[h];
        const float f[4] = {t.x, t.y, t.z, t.w};
        TO* to = out + (size_t)(tok0 + r[h]) * p.ldo + col;
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (col + i < p.feats) to[i] = from_float<TO>(f[i] + (bias ? bias[col + i] : 0.f));
      }
    }
    // (what the others have here has been read before it is used; the stores need not have arrived)
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if (CG == 2) g8_cluster_sync();
  if (warp == G8_EPI_WARPS + 1) {
    tc_fence_after();
    if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_slot), "r"((unsigned)G8_COLS) : "memory");
    else tc_dealloc(tmem_slot, G8_COLS);
  }
  if constexpr (EPI == G8_GATED) {
    // (the whole CTA: a thread to 8 of k)
    int looked = n_near;
    const bool all = looked > G8_NEAR || n_items > 1 << 25;
    // (out from here: between other launches the way over what follows, code that has to be fetched, was 0.3 to 1.0 us of each)
    if (looked == 0 && !all) return;
    double (*sums)[2] = reinterpret_cast<double (*)[2]>(base);
#pragma unroll 1
    for (int item = worker; item < n_items; item += n_workers) {
      if (all) {
        // Rounded numbers say where a scale may be that of a peak near the edge: 448 is then the largest one, or 224 of the higher scale.  One
        // block in ten is such and is looked at; what is far from the edge stays as it is.
        const G8Item q = g8_item(p, item, 0);
        const int row0 = row_x(q), col = q.ft * 128 + 4 * lane, n_rows = min(p.mrows, p.T - row0);
        __syncthreads();
        if (threadIdx.x == 0) n_near = 0;
        __syncthreads();
#pragma unroll 1
        for (int r = warp; r < n_rows; r += G8_THREADS / 32) {
          const unsigned char* of = (const unsigned char*)out + (size_t)(row0 + r) * p.ldo + col;
          unsigned most = 0;
#pragma unroll 1
          for (int e = 0; e < 4 && col + e < p.feats; e++) most = max(most, of[e] & 0x7fu);
          most = __reduce_max_sync(0xffffffffu, most);
          const unsigned byte = p.s_out[(size_t)(row0 + r) * p.lds_out + q.ft];
          if (lane == 0 && byte != 255u && (most == G8_448 ? byte >= 2 : most == G8_224 && byte >= 3)) near_rows[atomicAdd(&n_near, 1)] = r;
        }
        __syncthreads();
        looked = n_near;
      }
#pragma unroll 1
      for (int i = 0; i < looked; i++) {
        const G8Item q = g8_item(p, all ? item : near_rows[i] >> 7, 0);
        const long long row = row_x(q) + (int)(near_rows[i] & 127);
        const int col = q.ft * 128 + 4 * lane, there = min(4, p.feats - col);
        unsigned char *to = (unsigned char*)out + row * p.ldo + col, *scale = p.s_out + row * p.lds_out + q.ft;
        float v[4];
        unsigned most = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          v[e] = e < there ? fp8_value(to[e]) : 0.f;
          most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        // The scale is the one of at most 448, or twice that.  Those that count are the largest of the rounded ones; the edge is 448 of the lower.
        const bool higher = most < __float_as_uint(400.f);
        const unsigned low = *scale - higher;
        const unsigned edge = (low + 8) << 23 | 0x600000u;     // as float32
        // the gate's and up's sums of feature ``f`` in float64, as far as this warp has them
        const auto sums_of = [&](long long f, int first, int step, double& tg, double& tu) {
          tg = tu = 0.0;
#pragma unroll 1
          for (int k = first; k < p.K; k += step) {
            float a[8], b[8], d[8];
            double sg = 0.0, su = 0.0;
            g8_eight(a, p.x + row * p.ldx + k, p.K - k);
            g8_eight(b, p.w + f * p.ldw + k, p.K - k);
            g8_eight(d, p.w + (p.feats + f) * p.ldw + k, p.K - k);
            const int block = k >> 7;
            const unsigned sx = p.sx[row * p.ldsx + block];
#pragma unroll
            for (int j = 0; j < 8; j++) {
              sg += a[j] * b[j];                               // (a product of two such numbers has 8 bits)
              su += a[j] * d[j];
            }
            tg += sg * g8_scaled(sx, p.sw[f * p.ldsw + block]);
            tu += su * g8_scaled(sx, p.sw[(p.feats + f) * p.ldsw + block]);
          }
          for (int d = 16; d; d >>= 1) {
            tg += __shfl_xor_sync(0xffffffffu, tg, d);
            tu += __shfl_xor_sync(0xffffffffu, tu, d);
          }
        };
        const auto bias_of = [&](long long f) { return bias ? (double)bias[f] : 0.0; };
        // First whether the block is over the edge, the whole CTA for each feature that may say so
        bool over = false;
#pragma unroll 1
        for (int e = 0; e < 4 && !over; e++) {
          const float of = e == 0 ? v[0] : e == 1 ? v[1] : e == 2 ? v[2] : v[3];
#pragma unroll 1
          for (unsigned c = __ballot_sync(0xffffffffu, (__float_as_uint(of) & 0x7fffffffu) == most); c && !over; c &= c - 1) {
            const long long f = q.ft * 128 + 4 * (__ffs(c) - 1) + e;
            double tg, tu;
            sums_of(f, 8 * threadIdx.x, 8 * G8_THREADS, tg, tu);
            __syncthreads();                                   // (what the sums before were is no longer read)
            if (lane == 0) {
              sums[warp][0] = tg;
              sums[warp][1] = tu;
            }
            __syncthreads();
            tg = bias_of(f);
            tu = bias_of(p.feats + f);
#pragma unroll 1
            for (int j = 0; j < G8_THREADS / 32; j++) {
              tg += sums[j][0];
              tu += sums[j][1];
            }
            // (the float32 activation is 6 units of 2^-23 off at most, its arguments' rounding makes 1, and |a'| g / 2 for the gate, 10 for gelu at
            // -3: 30 units at 1.75.  Only nearer than that, and for deeper gates, float64 has to say, 0.5 us)
            const int off = (int)(__float_as_uint(fp8_gated((float)tg, (float)tu, p.act)) & 0x7fffffffu) - (int)edge;
            over = tg > -3.0 && abs(off) > 32 ? off > 0 : fabs(fp8_gated_64(tg, tu, p.act)) > (double)__uint_as_float(edge);
          }
        }
        if (over == higher) continue;
        // Its scale changes.  Numbers that are among e4m3's smallest, 2^-9 apart, at one of the scales are made again, a warp to each: the rounded
        // ones have lost, or would be rounded twice.  (Zeros of the lower scale stay; others are as far apart for their size at both.)
        float* fresh = reinterpret_cast<float*>(sums + G8_THREADS / 32);
        const double unit = g8_scaled(254 - low - over, 127);
        const float by = over ? 0.5f : 2.f;
        int turn = warp;
        bool made[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          made[e] = e < there && fabsf(v[e]) < 0.03125f && (!over || v[e] != 0.f);
          v[e] *= by;
#pragma unroll 1
          for (unsigned c = __ballot_sync(0xffffffffu, made[e]); c; c &= c - 1) {
            if (turn-- != 0) continue;
            turn = G8_THREADS / 32 - 1;
            const int at = 4 * (__ffs(c) - 1) + e;
            const long long f = q.ft * 128 + at;
            double tg, tu;
            sums_of(f, 8 * lane, 8 * 32, tg, tu);
            if (lane == 0) fresh[at] = (float)(fp8_gated_64(tg + bias_of(f), tu + bias_of(p.feats + f), p.act) * unit);
          }
        }
        __syncthreads();                                       // all have read the row
        if (warp == 0) {
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (made[e]) v[e] = fresh[4 * lane + e];
          const unsigned w = fp8_pack4(v[0], v[1], v[2], v[3]);
          for (int e = 0; e < there; e++) to[e] = (unsigned char)(w >> 8 * e);
          if (lane == 0) *scale = (unsigned char)(low + over);
        }
        __syncthreads();                                       // (the block may come again, and all have to see it alike)
      }
      if (!all) break;
    }
  }
}

// ------------------------------------------------------------------------------------ host
static int* g_status[64];
static int* status_word() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  if (!g_status[dev]) {
    int* ptr = nullptr;
    if (cudaMalloc(&ptr, sizeof(int)) != cudaSuccess) return nullptr;
    cudaMemset(ptr, 0, sizeof(int));
    g_status[dev] = ptr;
  }
  return g_status[dev];
}

static int up(int a, int b) { return (a + b - 1) / b; }

template <int EPI, typename TO, int CG>
static int g8_launch(const CUtensorMap& map_w, const CUtensorMap& map_x, const float* bias, void* out, const G8Params& p, int* status,
                     int ctas, size_t smem, cudaStream_t stream) {
  static bool allowed[64];                     // by device; all shared memory that a launch may ask for
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return QD_ERR_UNSUPPORTED;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(gemm_fp8_kernel<EPI, TO, CG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             G8_MAX_SMEM) != cudaSuccess)
      return (int)cudaGetLastError();
    allowed[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(G8_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = EPI == G8_SHARED ? p.splits : CG;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = qd_pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&cfg, gemm_fp8_kernel<EPI, TO, CG>, map_w, map_x, bias, (TO*)out, p, status);
  return qd_last_error();
}

// How many clusters of ``n`` CTAs run at a time: they lie within a group of multiprocessors, whose sizes need not be a multiple of theirs
// (of 148 multiprocessors 5 to a cluster leave some idle; a cluster too many doubles the time).
static int g8_clusters(int n, int sms) {
  static int known[64][9];                     // by device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    (void)cudaGetLastError();
    return sms / (n + 1);
  }
  if (known[dev][n]) return known[dev][n];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n * 148);
  cfg.blockDim = dim3(G8_THREADS);
  cfg.dynamicSmemBytes = G8_MAX_SMEM;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = n;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int got = 0;
  if (cudaFuncSetAttribute(gemm_fp8_kernel<G8_SHARED, bf16, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, G8_MAX_SMEM) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&got, gemm_fp8_kernel<G8_SHARED, bf16, 1>, &cfg) != cudaSuccess || got < 1) {
    (void)cudaGetLastError();
    got = sms / (n + 1);
  }
  return known[dev][n] = got;
}

extern "C" int qd_gemm_fp8_clusters(int n, int sms) { return n >= 1 && n <= 8 ? g8_clusters(n, sms) : 0; }

// How a product is cut: *cg CTAs to a tile of tokens, *bn rows of W to a tile, K in *splits shares (of a cluster).
//
// The one of the least estimate, in clocks of 1.9 GHz: a worker's rounds over its tiles times its blocks of 128 k, a block being the longest of
// its MMAs, its bytes into shared memory (70 a clock) and what one costs anyway; W's way from memory, the longer of both and half of the other;
// an epilogue; a cluster's joining and its CTAs.  Fitted to 6,866 times of 154 shapes (1 to 2,048 tokens, 102 to 20,000 features, 111 to 18,944 of
// k) in captured graphs on a B200, 5 % rms; the choices take 2.5 % longer than the best of all cuts on average.  Some of them, us, the chosen
// one and the best of the other kind (without shares where it has some, one CTA where it has two, and the other way round):
//   1 x 2,048 x 11,008      1 CTA, 192 rows, 8 shares   9.2   32 rows, 1 share   23.2
//   23 x 4,608 x 3,584      1 CTA, 192 rows, 4 shares   8.1   64 rows, 1 share   10.4
//   256 x 3,584 x 18,944    1 CTA, 224 rows, 4 shares  23.9   64 rows, 1 share   39.4
//   2,048 x 3,584 x 3,584   2 CTAs, 224 rows           23.6   1 CTA, 224 rows    24.4
//   2,048 x 3,584 x 18,944  2 CTAs, 224 rows          128.2   1 CTA, 208 rows   134.8   (under the power limit; alone 106.9 and 113.1)
extern "C" int qd_gemm_fp8_plan(int T, int N, int K, int epi, int out_dtype, int sms, int* cg_out, int* bn_out, int* splits_out) {
  epi &= 255;
  if (T <= 0 || N <= 0 || K <= 0 || sms < 2) return 0;
  const int kb = up(K, FP8_BLOCK), most = epi == G8_STORE && out_dtype == QD_F32 ? G8_MAX_FLOAT_BN : 256, feats = epi == G8_GATED ? N / 2 : N;
  const double dram = (double)N * K / 5290.0;
  double best = 0;
  for (int cg = 1; cg <= (T > 128 ? 2 : 1); cg++) {
    const int n_tt = up(T, 128 * cg), mrows = up(up(T, cg * n_tt), 8) * 8;
    for (int bn = epi == G8_GATED ? 256 : 32; bn <= most; bn += cg == 2 ? 32 : 16) {
      const long long tiles = (long long)up(feats, epi == G8_GATED ? bn / 2 : bn) * n_tt;
      const double block = fmax(fmax(2.37 * bn, (mrows + bn / cg) * 128 / 70.0), cg == 2 ? 542.0 : 486.0);
      for (int splits = 1; splits <= (epi == G8_GATED || cg == 2 || bn % 32 ? 1 : 8) && splits <= kb; splits++) {
        if (splits > 1 && tiles > g8_clusters(splits, sms)) break;
        const long long workers = sms / cg, rounds = splits > 1 ? 1 : (tiles + workers - 1) / workers;
        const double work = (double)rounds * up(kb, splits) * block + (rounds - 1) * 7.7 * bn;
        double cost = fmax(work, dram) + 0.505 * fmin(work, dram) + (0.214 * mrows + 7.7) * bn;
        if (splits > 1) cost += 70.0 * splits + 4830.0 * tiles * splits / sms;
        if (best == 0 || cost < best) { best = cost; *cg_out = cg; *bn_out = bn; *splits_out = splits; }
      }
    }
  }
  return 1;
}

// rows x cols bytes, rows ``ld`` bytes apart; boxes of box_rows rows of 128 bytes, 128-byte swizzle, zeros outside
static bool g8_make_map(CUtensorMap* map, const void* base, long long rows, long long cols, int box_rows, long long ld) {
  TcEncodeFn fn = tc_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {128u, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// X [T, K] and W [N, K] e4m3, rows ``ldx`` and ``ldw`` bytes apart (multiples of 16, as the addresses), with scales sx and sw, rows
// ``ldsx`` and ``ldsw`` bytes apart (multiples of 4, as the addresses).  epi 0: out [T, N] = X W^T (+ bias
// float32 [N]), bfloat16 or float32, rows ``ldo`` apart; ``splits`` > 1: K shared by clusters of so many CTAs (up to 8), a tile to each.
// epi 2 (+ 256 * QD_ACT_*): W [2F, K] the gate's rows, then up's; out e4m3 [T, F] = act(X Wg^T) * (X Wu^T), rows ``ldo`` bytes apart
// (a multiple of 4), and its scales s_out, rows ``lds_out`` apart.  ``cg``: CTAs to a tile of tokens, 1 (up to 128) or 2 (up to 256);
// ``bn``: rows of W to a tile, a multiple of 16 (of 32 for pairs and clusters) from 32 to 256 (256 for epi 2).  ``resident``: W and sw are
// written by nothing that may still run on the stream; they are then asked for before the kernels before this one have ended.
extern "C" int qd_gemm_fp8(const void* W, long long ldw, const void* sw, long long ldsw, const void* X, long long ldx, const void* sx,
                           long long ldsx, const float* bias, void* out, int out_dtype, long long ldo, void* s_out, long long lds_out,
                           int T, int N, int K, int cg, int bn, int splits, int epi, int resident, int sms, cudaStream_t stream) {
  if (T <= 0 || N <= 0) return 0;
  const int act = epi >> 8;
  epi &= 255;
  if (T > (1 << 30) || N > (1 << 30) || K <= 0 || K > (1 << 30) || ldx % 16 || ldw % 16 || ldx < K || ldw < K || (cg != 1 && cg != 2) ||
      bn < 32 || bn > 256 || bn % (cg == 2 || splits > 1 ? 32 : 16) || splits < 1 || splits > 8 || sms < 2 || !out)
    return QD_ERR_UNSUPPORTED;
  if ((((uintptr_t)W | (uintptr_t)X) & 15) || (((uintptr_t)sw | (uintptr_t)sx) & 3) || ldsw % 4 || ldsx % 4) return QD_ERR_UNSUPPORTED;
  if (epi == G8_GATED ? ((N & 1) || bn != 256 || splits != 1 || !s_out || ldo % 4 || (act != QD_ACT_SILU && act != QD_ACT_GELU_TANH))
                      : epi != G8_STORE)
    return QD_ERR_UNSUPPORTED;
  G8Params p;
  p.act = act; p.resident = resident; p.T = T; p.N = N; p.K = K; p.bn = bn; p.splits = splits; p.ldo = ldo;
  p.sx = (const unsigned char*)sx; p.sw = (const unsigned char*)sw; p.ldsx = ldsx; p.ldsw = ldsw;
  p.doubt = g8_doubt(K); p.x = (const unsigned char*)X; p.w = (const unsigned char*)W; p.ldx = ldx; p.ldw = ldw;
  p.s_out = (unsigned char*)s_out; p.lds_out = lds_out;
  p.kb_total = up(K, FP8_BLOCK);
  if (ldsx < p.kb_total || ldsw < p.kb_total) return QD_ERR_UNSUPPORTED;
  if (splits > p.kb_total || (splits > 1 && cg != 1) || (epi == G8_STORE && out_dtype == QD_F32 && bn > G8_MAX_FLOAT_BN)) return QD_ERR_UNSUPPORTED;
  p.feats = epi == G8_GATED ? N / 2 : N;
  p.n_tt = up(T, 128 * cg);
  p.mrows = up(up(T, cg * p.n_tt), 8) * 8;           // the tokens evenly over the token tiles and their CTAs
  p.n_ft = up(p.feats, epi == G8_GATED ? bn / 2 : bn);
  const long long items = (long long)p.n_ft * p.n_tt;
  if (items * splits > (1ll << 30)) return QD_ERR_UNSUPPORTED;
  const int workers = splits > 1 ? (int)items : (int)(items < sms / cg ? items : sms / cg);
  const int stage_bytes = (p.mrows + bn / cg) * 128;
  p.stages = G8_SMEM / stage_bytes;
  if (p.stages > G8_MAX_STAGES) p.stages = G8_MAX_STAGES;
  p.vec = !((uintptr_t)out & 15) && ldo % (epi == G8_GATED ? 16 : out_dtype == QD_F32 ? 4 : 8) == 0;
  // An MMA reads 128 rows of the last stage's tokens.  With fewer there are more stages, and the weights' stages behind them
  // hold at least 16 x 32 rows.
  const size_t smem = (size_t)p.stages * stage_bytes + G8_EPI_WARPS * G8_STAGE_ROWS + 1024;
  // (a share's sums lie where the stages were: at most 128 KB, and with few rows or features the stages are as many)
  if (splits > 1 && (size_t)p.mrows * bn * 4 > (size_t)p.stages * stage_bytes) return QD_ERR_UNSUPPORTED;
  int* status = status_word();
  CUtensorMap map_w, map_x;
  const int box = epi == G8_GATED || cg == 2 ? bn / 2 : bn;
  if (!status || !g8_make_map(&map_w, W, N, K, box, ldw) || !g8_make_map(&map_x, X, T, K, p.mrows, ldx)) return QD_ERR_UNSUPPORTED;
#define GO(E, TO)                                                                                                      \
  return cg == 2 ? g8_launch<E, TO, 2>(map_w, map_x, bias, out, p, status, 2 * workers, smem, stream)                   \
                 : g8_launch<E, TO, 1>(map_w, map_x, bias, out, p, status, workers, smem, stream)
#define GO1(E, TO) return g8_launch<E, TO, 1>(map_w, map_x, bias, out, p, status, workers * splits, smem, stream)
  if (epi == G8_GATED) GO(G8_GATED, unsigned char);
  if (splits > 1 && out_dtype == QD_BF16) GO1(G8_SHARED, bf16);
  if (splits > 1 && out_dtype == QD_F32) GO1(G8_SHARED, float);
  if (out_dtype == QD_BF16) GO(G8_STORE, bf16);
  if (out_dtype == QD_F32) GO(G8_STORE, float);
#undef GO
#undef GO1
  return QD_ERR_UNSUPPORTED;
}

// 0 if no bounded wait of this library's kernel has run out on the current device (1: producer, for a free stage; 2: MMAs, for
// data; 3: MMAs, for a drained accumulator; 4: epilogue; 5: MMAs, for scales; 6: scales, for a free buffer).  Synchronises the device.
QD_DEFINE_WAIT_PROBE(qd_gemm_fp8_wait_probe, tc_wait(bar, 0, dead, 0, poll_limit), status_word, 99)

extern "C" int qd_gemm_fp8_status() {
  int* status = status_word();
  if (!status) return -1;
  int v = 0;
  if (cudaMemcpy(&v, status, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) return -1;
  if (v) cudaMemset(status, 0, sizeof(int));
  return v;
}
