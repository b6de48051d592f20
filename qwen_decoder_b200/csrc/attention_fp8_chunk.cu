// Attention of portions of several requests' tokens over a paged cache in 8 bits (cache_fp8.cuh), causal, on the fifth-generation tensor cores:
//
//   z_k = scale 2^(s_k) (q . n_k),   p = softmax z over lo <= k <= pos,   out = sum_k p_k 2^(s_v) n_v
//
// A CTA takes 128 rows = (128 / gs) tokens x the gs query heads of one KV head, as attention_tc5.cu, and walks tiles of 128 keys.  The
// softmax, the weights P that go over the scores in tensor memory and the sums that stay there are that kernel's.  What 8 bits change:
//
// * Scores by kind::mxf8f6f4 with block scaling: the keys' numbers are the operand as they lie in the cache, the tensor cores apply a key's scale,
//   and nothing is converted.  Both operands have to be of 8 bits then, so a row of q is two of them: e4m3 numbers of q over the row's scale,
//   and of what their rounding left, over a sixteenth of it.  Together they are the bfloat16 number itself where it is above 2^-14 of the row's
//   largest, and off by 2^-23 of that below.  Two products of 128 features in 8 bits take the tensor cores as long as one of bfloat16.
// * Values become float16, an e4m3 number's scale over the tile's largest one, E, included, which is exact down to 2^-15 E: four warps take tiles from
//   where the copies leave them to where the product reads them.  P is float16 too, 2^(z + log E - reference): the product's sums are of
//   values as they are, and a row's sum of exponentials has a maximum of its own.  P is scaled so that 2^8 stands for the largest weight at the time its
//   reference was taken, and is off by 2^-11 of itself, or by 2^-33 of that weight where that is more.  Where a tile has a scale below 2^-15 of the
//   largest one up to it, values and P are bfloat16 as long as that is so, whose exponents take anything (E is 2^-60 of that largest one or more
//   then, so that no exponential is lost that a row's sum has).  (P in 8 bits would
//   be two numbers as q is, for every weight; this is 16 KB of values to a tile for all 128 rows.  Values to bfloat16, for every tile, took
//   twice the instructions: 2,048 tokens behind 6,144 420 us.)  These warps also bring the keys' scales to tensor memory.
// * A key or value that is no number has the scale 255.  The value becomes zeros, its key's scale 255, so that the score is none and
//   every row that sees it, and no other, is none.  Values behind the last row's position, which may be anything, become zeros.
// * Tiles of rows that would leave multiprocessors without work (a short portion behind a long history, the last round of a long one) share their
//   keys among CTAs, whose sums chunk_fp8_join_kernel adds up.
//
// With 28 + 4 heads of 128, 2,048 tokens behind 6,144 take 252 us, of which 125 are the products at the rate of a library's; a tile of 128 x 128 takes some
// 2,200 cycles, in which the softmax warps never wait: 1,024 are the exponentials' (16 a cycle), the rest what comes before and behind them (scores
// from tensor memory, maxima, the other half's maximum, weights back).  37 tokens behind 32,000 take 41 us, of which 10 are their products': three tiles of rows,
// the last of them one token's, in 12 shares each.  512 tokens of three requests behind 655 at most, 16 + 2 heads: 16.7 us, of which the launch and the way to
// the first scores (rows, q's operands) are 6.
//
// Warps: 0..7 softmax (two threads to a row: halves of the keys and of the columns), 8 and 9 copies of keys and values, 10 MMAs, 11 scales,
// 12..15 values.
// Slot i (i = -2 .. n - 1; stage (i + 2) % 3) holds the keys of tile i + 2 with their scales and the values of tile i: what the MMA warp
// reads in its step i, behind one barrier.  Every wait on an mbarrier is bounded, as in attention_tc5.cu.
#include "attention_tc5.cuh"
#include "cache_fp8.cuh"
#include "entry_points.h"
#include "tc5_ops.cuh"

#include <cuda_fp16.h>
#include <math.h>

#define AC_SOFTMAX 256                 // threads
#define AC_VALUES 128                  // threads that convert
#define AC_THREADS 512
#define AC_STAGES 3
#define AC_META 256                    // requests whose token ranges are staged in shared memory
#define AC_ROWS 128
#define AC_KEYS 128
#define AC_GROW 7.0f                   // powers of two by which a row's maximum grows before it is followed
#define AC_IDLE 60                     // nanoseconds between two looks of a warp that is ahead, which the others' issue slots are better for
#define AC_TOP 8.0f                    // log2 of what stands for the maximum: below 2^15 in all, within float16
#define AC_WIDE 256u                   // beside a tile's largest scale: values and weights in bfloat16
#define AC_HOLES 512u                  // and: some of the values are nobody's or no numbers
#define AC_AHEAD 8                     // tiles of whose scales something is kept
#define AC_SPREAD 15                   // powers of two between scales up to which they are float16
#define AC_DEEP 60                     // and what a tile's largest one is taken to be below the largest of all at most
#define AC_NONE (-1e30f)               // the maximum of no scores
#define AC_REGS 128                    // a thread's at the launch; the host looks that it is so
#define AC_REGS_SOFTMAX 184            // 2 x 184 + 56 + 88 = 4 x 128
#define AC_REGS_ISSUE 56
#define AC_REGS_VALUES 88
static_assert(2 * AC_REGS_SOFTMAX + AC_REGS_ISSUE + AC_REGS_VALUES <= 4 * AC_REGS, "registers of the block's four groups of warps");

struct AcParams {
  const bf16* q; long long ldq;
  bf16* out; long long ldo;
  const unsigned char* pages; long long page_bytes; int n_pages;
  const int* table; int max_blocks;
  const int *cu, *start;
  int R, rows, H, G, ps, ps_shift, window, tok_tile;      // ps_shift: log2 of ps, or -1
  float scale_log2e;
  // Pairs of a tile of rows and a KV head, the longest first; the ones before ``whole`` are a CTA's each, those behind it ``shares`` CTAs', which
  // leave their sums: [pair][share][128][HD], [pair][share][128][4]: reference, maximum of scores, sum of exponentials
  int tiles, whole, shares;
  float *part_o, *part_s;
  int* status;
};

// A pair's rows: which request, which of its tokens (tiles numbered request by request)
struct AcRows { int r, tok0, n_tok, pos0; };
__device__ __forceinline__ AcRows ac_rows(const AcParams& p, const int* cu, const int* sp, int pair) {
  auto row_at = [&](int r) { return min(max(cu[r], 0), p.rows); };      // (no row is touched that is none, whatever the list says)
  const int b = p.tiles - 1 - (int)((unsigned)pair / (unsigned)p.G);
  AcRows a = {0, 0, 0, 0};
  int before = 0;
  for (; a.r < p.R; a.r++) {
    const int nt = (int)((unsigned)(max(row_at(a.r + 1) - row_at(a.r), 0) + p.tok_tile - 1) / (unsigned)p.tok_tile);
    if (b < before + nt) break;
    before += nt;
  }
  if (a.r < p.R) {                     // (else: no rows)
    a.tok0 = row_at(a.r) + (b - before) * p.tok_tile;
    a.n_tok = min(p.tok_tile, row_at(a.r + 1) - a.tok0);
    a.pos0 = sp[a.r] + (b - before) * p.tok_tile;
  }
  return a;
}

__device__ __forceinline__ int ac_key_lo(const AcParams& p, int pos) { return p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0; }
// x: byte of a row, y: row of a page, z: page
__device__ __forceinline__ void ac_load_3d(void* dst, const CUtensorMap* map, int y, int z, unsigned long long* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(tc_smem(dst)), "l"(map), "r"(tc_smem(bar)), "r"(0), "r"(y), "r"(z) : "memory");
}
// D[128 x 128] (+)= A[128 x 32] B[128 x 32]^T of e4m3 numbers with a scale to each row of A and of B: A in tensor memory, four neighbouring k a column
__device__ __forceinline__ void ac_mma_scaled(unsigned d, unsigned a, unsigned desc_lo, unsigned desc_hi, unsigned idesc, unsigned sa, unsigned sb,
                                              unsigned accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 d;\n setp.ne.b32 p, %7, 0;\n mov.b64 d, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], [%1], d, %4, [%5], [%6], p;\n}\n"
      ::"r"(d), "r"(a), "r"(desc_lo), "r"(desc_hi), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void ac_st4(unsigned addr, unsigned a, unsigned b, unsigned c, unsigned d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// whether the phase with this parity has completed, by one look
__device__ __forceinline__ bool ac_done(unsigned long long* bar, unsigned parity) {
  unsigned ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok) : "r"(tc_smem(bar)), "r"(parity) : "memory");
  return ok;
}
__device__ __forceinline__ unsigned ac_halves(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
// 2^x, subnormal numbers included
__device__ __forceinline__ float ac_power(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two float32 numbers in one register pair
__device__ __forceinline__ unsigned long long ac_two(float a, float b) {
  unsigned long long v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 ac_both(unsigned long long v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ unsigned long long ac_fma(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ unsigned long long ac_add(unsigned long long a, unsigned long long b) {
  unsigned long long v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
// two e4m3 numbers times two float16 numbers
__device__ __forceinline__ unsigned ac_f16x2(unsigned short two, unsigned f) {
  unsigned h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
  asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(h) : "r"(f));
  return h;
}
// two e4m3 numbers
__device__ __forceinline__ float2 ac_values(unsigned short two) {
  unsigned h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// two e4m3 numbers times f as bfloat16
__device__ __forceinline__ unsigned ac_bf16x2(unsigned short two, float f) {
  const float2 v = ac_values(two);
  return at_pack(v.x * f, v.y * f);
}

template <int HD>
__global__ void __launch_bounds__(AC_THREADS, 1) chunk_fp8_kernel(const __grid_constant__ CUtensorMap map, const AcParams p) {
  constexpr int KQ = AC_KEYS / 2, DH = HD / 2, NS = AC_STAGES;
  constexpr int TILE8 = AC_KEYS * HD, TILE16 = 2 * TILE8;           // bytes of a tile in 8 bits, in 16
  constexpr int BOX = 16 * HD;
  // tensor memory: two buffers of scores and weights, the sums, q's two operands of HD / 4 columns, their scales, the keys' scales
  constexpr unsigned TMEM_COLS = 512, T_O = 2 * AC_KEYS, T_Q = 3 * AC_KEYS, T_SA = 448, T_SB = 456;
  // rows of 128 (64) bytes with the 128-byte (64-byte) swizzle, groups of 8 rows 1024 (512) bytes apart
  constexpr unsigned K_DESC_HI = HD == 128 ? AT_DESC_HI : (unsigned)(512 >> 4) | (1u << 14) | (4u << 29);
  extern __shared__ __align__(16) unsigned char smem_raw[];
  unsigned char* base = smem_raw + ((1024 - (tc_smem(smem_raw) & 1023)) & 1023);
  unsigned char* k_s = base;                        // NS stages of keys
  unsigned char* v8_s = k_s + NS * TILE8;           // NS stages of values as they come
  unsigned char* v_s = v8_s + NS * TILE8;           // NS stages of values in 16 bits
  __shared__ unsigned long long full[NS], empty[NS], v8_full[NS], v8_empty[NS], s_full[2], p_full[2], o_done, o_last, q_full;
  __shared__ float mx_s[2][2][AC_ROWS], l_s[2][AC_ROWS];
  __shared__ unsigned sa_s[AC_ROWS];
  // of a tile: its values' largest scale with AC_WIDE and AC_HOLES, its keys' scales, by what its values are multiplied (two float16 numbers; a
  // float32 number where they become bfloat16; 0: nobody's)
  __shared__ unsigned tile_s[AC_AHEAD];
  __shared__ __align__(16) unsigned key_s[AC_AHEAD][AC_KEYS / 4], factor_s[AC_AHEAD][AC_KEYS];
  __shared__ unsigned tmem_slot;
  __shared__ int dead;
  __shared__ int cu_s[AC_META + 1], sp_s[AC_META + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    dead = 0;
    for (int s = 0; s < NS; s++) {
      // (a warp's threads arrive by one of them)
      tc_bar_init(&full[s], 1 + AC_VALUES / 32);
      tc_bar_init(&empty[s], 1);
      tc_bar_init(&v8_full[s], 2);
      tc_bar_init(&v8_empty[s], AC_VALUES / 32);
    }
    for (int s = 0; s < 2; s++) { tc_bar_init(&s_full[s], 1); tc_bar_init(&p_full[s], AC_SOFTMAX / 32); }
    // (o_last: the last product has no scores behind it by which its phase of o_done would be known)
    tc_bar_init(&o_done, 1); tc_bar_init(&o_last, 1);
    tc_bar_init(&q_full, AC_SOFTMAX / 32);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 10) tc_alloc(&tmem_slot, TMEM_COLS);
  pdl_wait();
  const bool staged = p.R < AC_META;
  if (staged)
    for (int i = threadIdx.x; i <= p.R; i += AC_THREADS) {
      cu_s[i] = p.cu[i];
      sp_s[i] = i < p.R ? p.start[i] : 0;
    }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = tmem_slot;

  // ---- which rows, and which share of their keys
  const int behind = (int)blockIdx.x - p.whole, pair = behind < 0 ? blockIdx.x : p.whole + (unsigned)behind / (unsigned)p.shares;
  const int share = behind < 0 ? 0 : (unsigned)behind % (unsigned)p.shares;
  const int shares = behind < 0 ? 1 : p.shares;
  const int g = (unsigned)pair % (unsigned)p.G, gs = (unsigned)p.H / (unsigned)p.G;
  const AcRows rows = ac_rows(p, staged ? cu_s : p.cu, staged ? sp_s : p.start, pair);
  const bool idle = rows.r == p.R;
  const int r = rows.r, tok0 = rows.tok0, n_tok = rows.n_tok, pos0 = rows.pos0;
  const int key_hi = pos0 + n_tok, key_lo = ac_key_lo(p, pos0);
  // of the tiles from the first row's first key to the last row's last, this share's
  const int t0 = key_lo / AC_KEYS, tn = idle ? 0 : max((key_hi + AC_KEYS - 1) / AC_KEYS - t0, 0);
  // (2^24 tiles and 64 shares at most: 32 bits, whose quotients are a third of the way)
  const int kt_lo = t0 + (int)((unsigned)(tn * share) / (unsigned)shares), n_kt = t0 + (int)((unsigned)(tn * (share + 1)) / (unsigned)shares) - kt_lo;
  const int* table = p.table + (long long)(idle ? 0 : r) * p.max_blocks;
  // of a key: its page's entry in the table, for whoever needs it a tile later (keys that are none: any page will do); the page; the place in it
  auto entry_at = [&](int key) {
    const int block = p.ps_shift >= 0 ? key >> p.ps_shift : key / p.ps;
    return key < key_hi && block < p.max_blocks ? table[block] : 0;
  };
  auto page_of_entry = [&](int entry) { return min(max(entry, 0), p.n_pages - 1); };
  auto offset_of = [&](int key) { return p.ps_shift >= 0 ? key & (p.ps - 1) : key % p.ps; };

  if (warp < AC_SOFTMAX / 32) {
    // ------------------------------------------------------------------ softmax: two threads to a row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AC_REGS_SOFTMAX));
    const int row = (warp & 3) * 32 + lane, h = warp >> 2;          // row: also the lane of tensor memory
    const int t = (unsigned)row / (unsigned)gs, hh = row - t * gs;
    const bool ok = !idle && t < n_tok;
    const int pos = pos0 + t, lo = ac_key_lo(p, pos);
    const unsigned t_lane = tmem + ((unsigned)((warp & 3) * 32) << 16);
    {
      // this thread's half of the row of q as e4m3 numbers over the row's scale, and what that left over a sixteenth of it
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (long long)(tok0 + t) * p.ldq + (long long)(g * gs + hh) * HD + h * DH);
      uint4 w[DH / 8];
      unsigned peak = 0;                             // (magnitudes order as their bits do)
#pragma unroll
      for (int i = 0; i < DH / 8; i++) {
        w[i] = ok ? src[i] : make_uint4(0, 0, 0, 0);
        const unsigned x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int j = 0; j < 4; j++) peak = max(peak, max(x[j] << 16 & 0x7fffffffu, x[j] & 0x7fff0000u));
      }
      mx_s[0][h][row] = __uint_as_float(peak);
      asm volatile("bar.sync 1, %0;" ::"n"(AC_SOFTMAX) : "memory");
      unsigned byte = fp8_scale_byte(max(peak, __float_as_uint(mx_s[0][h ^ 1][row])));
      byte = max(byte, 5u);                          // (a sixteenth of it is a scale as well)
      const float inv = fp8_inverse(byte);
      unsigned big[DH / 4], small[DH / 4];
#pragma unroll
      for (int i = 0; i < DH / 4; i++) {
        const unsigned* x = &w[i / 2].x + 2 * (i & 1);
        const float v0 = __uint_as_float(x[0] << 16) * inv, v1 = __uint_as_float(x[0] & 0xffff0000u) * inv;
        const float v2 = __uint_as_float(x[1] << 16) * inv, v3 = __uint_as_float(x[1] & 0xffff0000u) * inv;
        big[i] = fp8_pack4(v0, v1, v2, v3);
        const float2 b01 = ac_values((unsigned short)big[i]), b23 = ac_values((unsigned short)(big[i] >> 16));
        small[i] = fp8_pack4((v0 - b01.x) * 16.f, (v1 - b01.y) * 16.f, (v2 - b23.x) * 16.f, (v3 - b23.y) * 16.f);
      }
#pragma unroll
      for (int i = 0; i < DH / 4; i += 8) {
        unsigned x[8], y[8];
#pragma unroll
        for (int j = 0; j < 8; j++) { x[j] = big[i + j]; y[j] = small[i + j]; }
        tc_st8(t_lane + T_Q + h * (DH / 4) + i, x);
        tc_st8(t_lane + T_Q + HD / 4 + h * (DH / 4) + i, y);
      }
      if (h == 0) sa_s[row] = byte;
      asm volatile("bar.sync 1, %0;" ::"n"(AC_SOFTMAX) : "memory");
      if (h == 0) {                                  // lane l, column c: the scale of row 32 c + l, in every quarter of the lanes
        unsigned a[4];
#pragma unroll
        for (int c = 0; c < 4; c++) a[c] = sa_s[32 * c + lane];
        ac_st4(t_lane + T_SA, a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int c = 0; c < 4; c++) a[c] = a[c] == 255u ? 255u : a[c] - 4u;
        ac_st4(t_lane + T_SA + 4, a[0], a[1], a[2], a[3]);
      }
      tc_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) tc_arrive(&q_full);
    }
    // m: the maximum that this row's weights and output refer to; z: of its scores so far, which the sum of its exponentials refers to
    float m = -INFINITY, z = AC_NONE, l = 0.f;
    const int free_hi = pos0 + 1, free_lo = ac_key_lo(p, key_hi - 1);       // keys that every row sees need no test
    bool ready = false;                  // the next tile's scores are there: looked at ahead, since the answer takes 200 to 300 cycles
    for (int j = 0; j < n_kt; j++) {
      const int tile_base = (kt_lo + j) * AC_KEYS, key_base = tile_base + h * KQ;
      if (!ready && !tc_wait_inline(&s_full[j & 1], (j >> 1) & 1, &dead) && lane == 0) atomicCAS(p.status, 0, 7);
      __syncwarp();                                  // (here and below: what follows is the whole warp's instruction)
      tc_fence_after();
      float sv[KQ];
      at_tmem_ld<KQ>(t_lane + (unsigned)(j & 1) * AC_KEYS + h * KQ, sv);
      const bool interior = tile_base >= free_lo && tile_base + AC_KEYS <= free_hi && p.scale_log2e > 0.f;
      if (!interior) {
        // of this thread's keys the first that the row sees, and how many
        const int from = max(lo - key_base, 0), many = ok ? max(pos - key_base - from + 1, 0) : 0;
#pragma unroll
        for (int i = 0; i < KQ; i++) sv[i] = (unsigned)(i - from) < (unsigned)many ? sv[i] * p.scale_log2e : -INFINITY;
      }
      float mx4[4] = {sv[0], sv[1], sv[2], sv[3]};   // (one chain of 64 would be four cycles each)
#pragma unroll
      for (int i = 4; i < KQ; i += 2) mx4[i / 2 & 3] = fmaxf(fmaxf(mx4[i / 2 & 3], sv[i]), sv[i + 1]);
      const float mul = interior ? p.scale_log2e : 1.0f;
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * mul;
      mx_s[j & 1][h][row] = mx;
      const unsigned tile = tile_s[j % AC_AHEAD];
      const float top = (float)((int)(tile & 255u) - 127);
      unsigned pk[KQ / 2];
      float sum;
      auto weigh = [&]() {                           // against the row's reference
        const float ref = (m == -INFINITY ? 0.f : m) - top - AC_TOP;
        sum = 0.f;
        if (tile & AC_WIDE) {
#pragma unroll
          for (int i = 0; i < KQ / 2; i++) {
            const float p0 = at_exp2(fmaf(sv[2 * i], mul, -ref)), p1 = at_exp2(fmaf(sv[2 * i + 1], mul, -ref));
            sum += p0 + p1;
            pk[i] = at_pack(p0, p1);
          }
        } else {                                     // (two numbers to an instruction: 2,048 tokens behind 6,144 283 -> 274 us)
          const unsigned long long by = ac_two(mul, mul), from = ac_two(-ref, -ref);
          unsigned long long two = 0;
#pragma unroll
          for (int i = 0; i < KQ / 2; i++) {
            const float2 x = ac_both(ac_fma(ac_two(sv[2 * i], sv[2 * i + 1]), by, from));
            const float p0 = at_exp2(x.x), p1 = at_exp2(x.y);
            two = ac_add(two, ac_two(p0, p1));
            pk[i] = ac_halves(p0, p1);
          }
          const float2 sums = ac_both(two);
          sum = sums.x + sums.y;
        }
      };
      ready = __all_sync(0xffffffffu, ac_done(&s_full[j & 1 ^ 1], (j + 1) >> 1 & 1));
      // Weights first, against the reference as it is; the other thread's maximum then seldom says that it has to move (the first tile's always).
      if (j > 0) weigh();
      asm volatile("bar.sync %0, 64;" ::"r"(3 + (warp & 3)) : "memory");       // the two warps of these rows
      const float z_tile = fmaxf(mx, mx_s[j & 1][h ^ 1][row]), m_tile = z_tile + top;       // of weights with the largest of the tile's scales
      // the row moves to a new reference only when its maximum has grown by more than AC_GROW (always from "no key yet"); both threads of a
      // row decide alike, and the warp acts together
      const bool grow = m_tile > m + AC_GROW;
      if (__any_sync(0xffffffffu, grow) || j == 0) {
        const float alpha = grow ? at_exp2(m - m_tile) : 1.0f;
        if (grow) m = m_tile;
        if (j > 0) {
          if (!tc_wait_inline(&o_done, (j - 1) & 1, &dead) && lane == 0) atomicCAS(p.status, 0, 8);
          __syncwarp();
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < DH; c += 32) {
            float ov[32];
            at_tmem_ld<32>(t_lane + T_O + h * DH + c, ov);
            unsigned ob[32];
#pragma unroll
            for (int i = 0; i < 32; i++) ob[i] = __float_as_uint(ov[i] * alpha);
            at_tmem_st<32>(t_lane + T_O + h * DH + c, ob);
          }
        }
        weigh();
      }
      const float z_new = fmaxf(z, z_tile);          // (the difference is bounded where there is a sum)
      l = fmaf(sum, at_exp2(fminf((m == -INFINITY ? 0.f : m) - top - z_new, 100.f)), l * at_exp2(z - z_new));
      z = z_new;
      at_tmem_st<KQ / 2>(t_lane + (unsigned)(j & 1) * AC_KEYS + h * KQ, pk);      // over the first half of this thread's own scores
      tc_fence_before();
      __syncwarp();
      if (lane == 0) tc_arrive(&p_full[j & 1]);
    }
    if (n_kt > 0) {
      if (!tc_wait_inline(&o_last, 0, &dead) && lane == 0) atomicCAS(p.status, 0, 9);
      __syncwarp();
      tc_fence_after();
    }
    l_s[h][row] = l;
    asm volatile("bar.sync 1, %0;" ::"n"(AC_SOFTMAX) : "memory");
    const float l_all = l + l_s[h ^ 1][row];
    if (shares > 1) {
      const long long at = (long long)behind * AC_ROWS + row;
      if (ok && h == 0) *reinterpret_cast<float4*>(p.part_s + 4 * at) = make_float4(m, z, l_all, 0.f);
      if (n_kt > 0) {
#pragma unroll 1
        for (int c = 0; c < DH; c += 32) {
          float ov[32];
          at_tmem_ld<32>(t_lane + T_O + h * DH + c, ov);      // the warp's access: rows without a token take part too
          if (ok) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(p.part_o + at * HD + h * DH + c + i) = make_float4(ov[i], ov[i + 1], ov[i + 2], ov[i + 3]);
          }
        }
      }
    } else {
      const float inv = l_all == 0.f ? 0.f : 1.f / l_all, up = ac_power(m - z);
      bf16* d = p.out + (long long)(tok0 + t) * p.ldo + (long long)(g * gs + hh) * HD + h * DH;
#pragma unroll 1
      for (int c = 0; c < DH; c += 32) {
        float ov[32];
        if (n_kt > 0) {
          at_tmem_ld<32>(t_lane + T_O + h * DH + c, ov);
        } else {                                     // (rows in front of the first position)
#pragma unroll
          for (int i = 0; i < 32; i++) ov[i] = 0.f;
        }
        if (ok) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 v;
            v.x = at_pack(ov[i] * inv * up, ov[i + 1] * inv * up);
            v.y = at_pack(ov[i + 2] * inv * up, ov[i + 3] * inv * up);
            v.z = at_pack(ov[i + 4] * inv * up, ov[i + 5] * inv * up);
            v.w = at_pack(ov[i + 6] * inv * up, ov[i + 7] * inv * up);
            *reinterpret_cast<uint4*>(d + c + i) = v;
          }
        }
      }
    }
  } else if (warp >= 12) {
    // ------------------------------------------------------------------ the keys' scales, and values to 16 bits
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AC_REGS_VALUES));
    // A warp's threads take 8 rows of 64 features at a time, four threads to a row: row r's 16 features in a block are where the swizzles put them,
    // and with the rows in this order (r and r ^ 5 side by side) neither the 16 bytes read nor the two times 16 written meet a conflict.
    const int q = lane >> 2, c = lane & 3, x = q & 1 ? (q >> 1) ^ 5 : q >> 1;
    const unsigned t_sb = tmem + ((unsigned)((warp & 3) * 32) << 16) + T_SB;
    constexpr int STEPS = AC_KEYS / 8 / 4 * (HD / 64);       // of a warp: 8 rows each, four groups of rows apart, one block of features after the other
    for (int i = -2; i < n_kt; i++) {
      const int s = (i + 2) % NS, j = i + 2;
      if (!tc_wait_inline(&empty[s], ((i + 2) / NS & 1) ^ 1, &dead, AC_IDLE) && lane == 0) atomicCAS(p.status, 0, 5);
      if (!tc_wait_inline(&v8_full[s], (i + 2) / NS & 1, &dead) && lane == 0) atomicCAS(p.status, 0, 6);
      __syncwarp();
      tc_fence_after();
      if (j < n_kt) {                                 // the keys' scales: lane l, column c has row 32 c + l's
        const unsigned char* k = reinterpret_cast<const unsigned char*>(key_s[j % AC_AHEAD]) + lane;
        ac_st4(t_sb + 4 * s, k[0], k[32], k[64], k[96]);
      }
      if (i >= 0) {
        const unsigned tile = tile_s[i % AC_AHEAD];
        const unsigned* factor = factor_s[i % AC_AHEAD] + (warp & 3) * 8 + x;
        const unsigned char* from = v8_s + s * TILE8 + ((warp & 3) * 8 + x) * HD;
        unsigned char* to = v_s + s * TILE16 + ((warp & 3) * 8 + x) * 128;
        const int a_at = ((2 * c) ^ x) << 4, b_at = ((2 * c + 1) ^ x) << 4;
        // (rolled: 2,048 tokens behind 6,144 276 -> 259 us at the time, with the code of both kinds of tile in one body; in two 274 to 294, with waits between the turns 267)
#pragma unroll 1
        for (int e0 = 0; e0 < STEPS; e0 += 4) {
          const int block = e0 / 4;
          uint4 v[4];
          unsigned f[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            v[e] = *reinterpret_cast<const uint4*>(from + e * 32 * HD + 16 * (HD == 128 ? (4 * block + c) ^ x : c ^ (x >> 1 & 3)));
            f[e] = factor[e * 32];
          }
          if (tile & (AC_WIDE | AC_HOLES)) {
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (f[e] == 0) v[e] = make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const unsigned* w = &v[e].x;
            unsigned o[8];
            if (tile & AC_WIDE) {
#pragma unroll
              for (int y = 0; y < 4; y++) {
                o[2 * y] = ac_bf16x2((unsigned short)w[y], __uint_as_float(f[e]));
                o[2 * y + 1] = ac_bf16x2((unsigned short)(w[y] >> 16), __uint_as_float(f[e]));
              }
            } else {
#pragma unroll
              for (int y = 0; y < 4; y++) {
                o[2 * y] = ac_f16x2((unsigned short)w[y], f[e]);
                o[2 * y + 1] = ac_f16x2((unsigned short)(w[y] >> 16), f[e]);
              }
            }
            unsigned char* row = to + block * (AC_KEYS * 128) + e * 32 * 128;
            *reinterpret_cast<uint4*>(row + a_at) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(row + b_at) = make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      tc_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        tc_arrive(&v8_empty[s]);
        tc_arrive(&full[s]);
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AC_REGS_ISSUE));
    if (warp < 10) {
      // ---------------------------------------------------------------- copies: a tile is eight boxes of 16 keys, each from its page
      const int which = warp - 8;                     // 0 keys, 1 values
      auto entry_of = [&](int j) { return lane < 8 && j < n_kt ? entry_at((kt_lo + j) * AC_KEYS + 16 * lane) : 0; };
      int next = entry_of(0);
      // slot i = u - 2 has the keys of tile u and the values of tile u - 2; a slot without is told without
      for (int u = 0; u < n_kt + 2; u++) {
        const int s = u % NS, j = which ? u - 2 : u;
        const bool have = j >= 0 && j < n_kt;
        unsigned long long* bar = which ? &v8_full[s] : &full[s];
        if (!tc_wait_inline(which ? &v8_empty[s] : &empty[s], (u / NS & 1) ^ 1, &dead, AC_IDLE)) {
          if (lane == 0) atomicCAS(p.status, 0, 1);
          break;                                      // (nobody waits any more, and no more copies are to arrive)
        }
        if (lane == 0) {
          if (have) tc_expect_tx(bar, TILE8);
          else tc_arrive(bar);
        }
        __syncwarp();
        if (have) {
          const int page = page_of_entry(next);
          next = entry_of(j + 1);
          if (lane < 8) {
            const int key = (kt_lo + j) * AC_KEYS + 16 * lane;
            ac_load_3d((which ? v8_s : k_s) + s * TILE8 + lane * BOX, &map, (which * p.G + g) * p.ps + offset_of(key), page, bar);
          }
        }
      }
    } else if (warp == 11) {
      // ---------------------------------------------------------------- scales, two tiles ahead of the values: a thread has four neighbouring keys'
      const unsigned char* scales = p.pages + (long long)2 * p.G * p.ps * HD + (long long)g * p.ps * 2;
      auto key_of = [&](int j) { return (kt_lo + j) * AC_KEYS + 4 * lane; };
      auto scales_at = [&](int j, int entry) {
        const int key = key_of(j);
        if (j >= n_kt || key >= key_hi) return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
        return __ldcg(reinterpret_cast<const uint2*>(scales + page_of_entry(entry) * p.page_bytes + 2 * offset_of(key)));
      };
      uint2 sc = n_kt > 0 ? scales_at(0, entry_at(key_of(0))) : make_uint2(0, 0);
      int entry = n_kt > 1 ? entry_at(key_of(1)) : 0;
      unsigned largest = 0;                           // of the values' scales so far
      for (int u = 0; u < n_kt + 2; u++) {
        const int s = u % NS;
        if (!tc_wait_inline(&v8_empty[s], (u / NS & 1) ^ 1, &dead, AC_IDLE) && lane == 0) atomicCAS(p.status, 0, 11);
        __syncwarp();
        if (u < n_kt) {
          const uint2 now = sc;
          sc = scales_at(u + 1, entry);
          entry = u + 2 < n_kt ? entry_at(key_of(u + 2)) : 0;
          // (four keys' bytes at a time, in little code: one warp goes through it, and the first scores of a launch wait for it)
          const unsigned values = __byte_perm(now.x, now.y, 0x7531), none = __vcmpeq4(values, ~0u);
          const int first = key_lo - key_of(u), last = key_hi - key_of(u);      // of the four, the ones that are somebody's
          const unsigned seen = values | (first <= 0 ? 0u : first >= 4 ? ~0u : ~(~0u << 8 * first)) | (last >= 4 ? 0u : last <= 0 ? ~0u : ~0u << 8 * last);
          const bool all = __all_sync(0xffffffffu, __vcmpeq4(seen, ~0u) == 0u);
          unsigned most = 0, least = 255;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const unsigned b = seen >> 8 * e & 255u;
            most = max(most, b + 1 & 255u);
            least = min(least, b);
          }
          most = __reduce_max_sync(0xffffffffu, most);
          least = __reduce_min_sync(0xffffffffu, least);
          if (most == 0) least = most = largest ? largest : 127u;            // (no value that is seen)
          else most--;
          largest = max(largest, most);
          most = max(most, largest - min(largest, (unsigned)AC_DEEP));
          const bool wide = largest - least > AC_SPREAD;
          unsigned f[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const unsigned b = seen >> 8 * e & 255u, down = most - min(b, most);
            f[e] = wide ? (127u - min(down, 127u)) << 23 : (down < 15 ? (15u - down) << 10 : 0x200u) * 0x10001u;
            if (b == 255u) f[e] = 0;
          }
          const int at = u % AC_AHEAD;
          key_s[at][lane] = __byte_perm(now.x, now.y, 0x6420) | none;          // (a value without a number: its key's score is none)
          *reinterpret_cast<uint4*>(&factor_s[at][4 * lane]) = make_uint4(f[0], f[1], f[2], f[3]);
          if (lane == 0) tile_s[at] = most | (wide ? AC_WIDE : 0u) | (all ? 0u : AC_HOLES);
        }
        __syncwarp();
        if (lane == 0) tc_arrive(&v8_full[s]);
      }
    } else if (warp == 10 && !idle) {
      // ---------------------------------------------------------------- MMAs: the whole warp goes through the tiles, one lane issues
      const bool one = tc_elect();
      const unsigned idesc_qk = (unsigned)(AC_KEYS >> 3) << 17 | 1u << 23 | (unsigned)(AC_ROWS >> 4) << 24;
      const unsigned idesc_f16 = (1u << 4) | (1u << 16) | ((unsigned)(HD >> 3) << 17) | ((unsigned)(AC_ROWS >> 4) << 24);
      const unsigned k_lo0 = at_desc_lo(tc_smem(k_s), 0), v_lo0 = at_desc_lo(tc_smem(v_s), AC_KEYS * 128);
      auto slot_ready = [&](int i) {
        if (!tc_wait_inline(&full[(i + 2) % NS], ((i + 2) / NS) & 1, &dead) && lane == 0) atomicCAS(p.status, 0, 2);
        __syncwarp();
      };
      auto scores = [&](int j) {
        const unsigned k_lo = k_lo0 + (unsigned)(j % NS) * (TILE8 >> 4);
#pragma unroll 1
        for (int part = 0; part < 2; part++)
#pragma unroll
          for (int k = 0; k < HD / 32; k++)
            ac_mma_scaled(tmem + (unsigned)(j & 1) * AC_KEYS, tmem + T_Q + part * (HD / 4) + k * 8, k_lo + k * 2, K_DESC_HI, idesc_qk,
                          tmem + T_SA + 4 * part, tmem + T_SB + 4 * (j % NS), part || k ? 1u : 0u);
      };
      if (n_kt > 0) {
        if (!tc_wait_inline(&q_full, 0, &dead) && lane == 0) atomicCAS(p.status, 0, 3);
#pragma unroll 1
        for (int j = 0; j < 2; j++) {                   // slots -2 and -1: the first two tiles' scores
          slot_ready(j - 2);
          tc_fence_after();
          if (one) {
            if (j < n_kt) scores(j);
            tc_commit(&empty[j % NS]);
            if (j < n_kt) tc_commit(&s_full[j & 1]);
          }
        }
        for (int j = 0; j < n_kt; j++) {
          const int s = (j + 2) % NS;
          slot_ready(j);
          if (!tc_wait_inline(&p_full[j & 1], (j >> 1) & 1, &dead) && lane == 0) atomicCAS(p.status, 0, 4);
          __syncwarp();
          tc_fence_after();
          const unsigned v_lo = v_lo0 + (unsigned)s * (TILE16 >> 4), idesc_pv = idesc_f16 | (tile_s[j % AC_AHEAD] & AC_WIDE ? 1u << 7 | 1u << 10 : 0u);
          if (one) {
#pragma unroll 2
            for (int k = 0; k < AC_KEYS / 16; k++)
              at_umma_ta(tmem + T_O, tmem + (unsigned)(j & 1) * AC_KEYS + (unsigned)(k + (k & 4)) * 8, v_lo + (unsigned)k * (2048 >> 4), AT_DESC_HI, idesc_pv,
                         (j > 0 || k > 0) ? 1u : 0u);
            tc_commit(j + 1 < n_kt ? &o_done : &o_last);
            if (j + 2 < n_kt) scores(j + 2);
            tc_commit(&empty[s]);
            if (j + 2 < n_kt) tc_commit(&s_full[j & 1]);
          }
        }
        // the last commit's arrival, and with it all before it
        if (!tc_wait_inline(&empty[(n_kt + 1) % NS], (n_kt + 1) / NS & 1, &dead) && lane == 0) atomicCAS(p.status, 0, 10);
      }
      __syncwarp();
    }
  }
  pdl_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if (dead)
    for (int i = 0; i < 1000; i++) __nanosleep(1000);        // copies on their way land in what is still this CTA's
  if (warp == 10) {
    tc_fence_after();
    tc_dealloc(tmem, TMEM_COLS);
  }
}

// The shares of the pairs behind ``whole``: a block to one's four rows, a thread to four features of one.
#define AC_JOIN_ROWS 4
template <int HD>
__global__ void __launch_bounds__(AC_JOIN_ROWS * HD / 4) chunk_fp8_join_kernel(const AcParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int behind = blockIdx.x / (AC_ROWS / AC_JOIN_ROWS), pair = p.whole + behind, g = pair % p.G, gs = p.H / p.G;
  const int row = blockIdx.x % (AC_ROWS / AC_JOIN_ROWS) * AC_JOIN_ROWS + threadIdx.x / (HD / 4), f = threadIdx.x % (HD / 4) * 4;
  const AcRows rows = ac_rows(p, p.cu, p.start, pair);
  const int t = row / gs, hh = row - t * gs;
  if (rows.r == p.R || t >= rows.n_tok) return;
  const long long first = (long long)behind * p.shares * AC_ROWS + row;
  float m = -INFINITY, z = AC_NONE, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  // (eight at a time are on their way: one after the other each is a trip to memory)
  for (int s0 = 0; s0 < p.shares; s0 += 8) {
    float4 st[8], v[8];
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const long long at = first + (s0 + u) * AC_ROWS;
      st[u] = v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s0 + u < p.shares) {
        st[u] = __ldcg(reinterpret_cast<const float4*>(p.part_s + 4 * at));
        v[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * HD + f));
      }
    }
#pragma unroll
    for (int u = 0; u < 8; u++) {
      if (s0 + u >= p.shares) break;
      const float z_new = fmaxf(z, st[u].y);
      l = fmaf(st[u].z, at_exp2(st[u].y - z_new), l * at_exp2(z - z_new));
      z = z_new;
      if (st[u].x == -INFINITY) continue;        // (no key, whose sums were not written, or no numbers)
      const float m_new = fmaxf(m, st[u].x), x = at_exp2(st[u].x - m_new), y = at_exp2(m - m_new);
      o.x = fmaf(v[u].x, x, o.x * y); o.y = fmaf(v[u].y, x, o.y * y); o.z = fmaf(v[u].z, x, o.z * y); o.w = fmaf(v[u].w, x, o.w * y);
      m = m_new;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l, up = ac_power(m - z);
  *reinterpret_cast<uint2*>(p.out + (rows.tok0 + t) * p.ldo + (long long)(g * gs + hh) * HD + f) =
      make_uint2(at_pack(o.x * inv * up, o.y * inv * up), at_pack(o.z * inv * up, o.w * inv * up));
}

// ------------------------------------------------------------------------------------ host
// the number of the first wait that ran out (made with the module, not by the first call, which may be a captured one)
static __device__ int ac_status;
static int* ac_status_word() {
  static int* words[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  if (!words[dev]) {
    void* w = nullptr;
    if (cudaGetSymbolAddress(&w, ac_status) != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    words[dev] = (int*)w;
  }
  return words[dev];
}

// How a launch is cut: pairs in all, those that are a CTA's each, the shares of the others
struct AcPlan { long long tiles, whole; int shares; };
// A CTA holds a multiprocessor.  What does not fill one round of them is shared out: all pairs where there are few, else those of the last
// round (the shortest), by as many shares as make its time least.  In tiles of keys (1.2 us each): rounds of what a share has, each with what a CTA
// costs besides, and with shares the launch that joins them and their sums' way through memory.  (With 28 + 4 heads: 18 tokens behind 4,000, 4 pairs
// of 32 tiles: 48.9 us whole, 22.7, 18.1, 16.7, 18.2 in 4, 8, 16, 24 shares; 37 behind 1,000, 12 of 9 tiles: 20.9, 17.5, 16.4, 16.9 in 1, 3, 5, 9;
// 512 behind 300 with 16 + 2 heads, 64 of 7: 18.5, 22.7 in 1, 2; behind 1,500, 64 of 16: 29.6, 28.4.)
#define AC_CTA 5.0
#define AC_JOIN 2.5
#define AC_SUMS (1.0 / 30)             // for each share
static AcPlan ac_plan(int T, int R, int H, int G, int window, int max_keys, int sms) {
  const int tok_tile = AC_ROWS / (H / G);
  const long long tiles = (T + tok_tile - 1) / tok_tile + (R > 1 ? R - 1 : 0), pairs = tiles * G;       // (of R requests at most)
  const long long seen = (long long)window + tok_tile, keys = window > 0 && seen < max_keys ? seen : max_keys;
  const double length = (double)keys / AC_KEYS;
  const long long rest = pairs % sms;
  AcPlan plan = {tiles, pairs, 1};
  double best = ceil(length) + AC_CTA;
  for (int s = 2; s <= 64 && rest && s <= length; s++) {
    const double time = (double)((rest * s + sms - 1) / sms) * (ceil(length / s) + AC_CTA) + AC_JOIN + (double)(rest * s) * AC_SUMS;
    if (time < best) { best = time; plan.shares = s; plan.whole = pairs - rest; }
  }
  return plan;
}

// float32 numbers of scratch memory that a launch takes
extern "C" long long qd_prefill_attention_fp8_scratch(int T, int R, int H, int G, int d, int window, int max_keys, int sms) {
  if (T < 1 || R < 1 || G < 1 || H < G) return 0;
  const AcPlan plan = ac_plan(T, R, H, G, window, max_keys, sms);
  return (plan.tiles * G - plan.whole) * plan.shares * AC_ROWS * (d + 4);
}
// and the kernels of it: where some of the pairs are shared out, the one that joins their shares, too
extern "C" int qd_prefill_attention_fp8_launches(int T, int R, int H, int G, int window, int max_keys, int sms) {
  if (T < 1 || R < 1 || G < 1 || H < G) return 0;
  const AcPlan plan = ac_plan(T, R, H, G, window, max_keys, sms);
  return plan.tiles * G > plan.whole ? 2 : 1;
}

template <int HD>
static int ac_launch(const CUtensorMap& map, const AcParams& p, cudaStream_t stream) {
  const size_t smem = 1024 + (size_t)AC_STAGES * 4 * AC_KEYS * HD;
  static bool allowed[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return QD_ERR_UNSUPPORTED;
  if (!allowed[dev]) {
    cudaFuncAttributes of;
    if (cudaFuncGetAttributes(&of, chunk_fp8_kernel<HD>) != cudaSuccess ||
        cudaFuncSetAttribute(chunk_fp8_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
      cudaGetLastError();
      return QD_ERR_UNSUPPORTED;
    }
    if (of.numRegs != AC_REGS) return QD_ERR_BUILD;            // (a split that adds up to more than the launch's waits for ever)
    allowed[dev] = true;
  }
  const unsigned behind = (unsigned)(p.tiles * p.G - p.whole);
  qd_launch(chunk_fp8_kernel<HD>, dim3(p.whole + behind * p.shares), dim3(AC_THREADS), smem, stream, map, p);
  if (behind) qd_launch(chunk_fp8_join_kernel<HD>, dim3(behind * (AC_ROWS / AC_JOIN_ROWS)), dim3(AC_JOIN_ROWS * HD / 4), 0, stream, p);
  return qd_last_error();
}

// q, out: bfloat16 [rows, H d], ``ldq`` and ``ldo`` apart; request r's tokens are rows cu[r] .. cu[r + 1] - 1, at most T of them in all, at the
// positions from start[r] on, its pages row r of table [R, max_blocks]; they see the keys up to their own, the last ``window`` of them if that is
// positive.  ``max_keys``: no request has more keys; only how the launch is cut goes by it.
extern "C" int qd_prefill_attention_fp8(const void* q, long long ldq, void* out, long long ldo, const void* pages, long long n_pages, const int* table,
                                        int max_blocks, const int* cu, const int* start, int R, int T, int rows, int H, int G, int d, int ps,
                                        float scale, int window, int max_keys, float* scratch, int sms, cudaStream_t stream) {
  if (T <= 0 || R <= 0) return 0;
  if (G < 1 || H < 1 || H % G || H / G > 16 || (d != 64 && d != 128) || ps < 16 || ps % 16 || n_pages < 1 || n_pages > 0x7fffffffll || max_blocks < 1 ||
      window < 0 || T > rows || G > 65535)
    return QD_ERR_UNSUPPORTED;
  if ((((uintptr_t)q | (uintptr_t)out | (uintptr_t)pages) & 15) || ldq % 8 || ldo % 8) return QD_ERR_UNSUPPORTED;
  int* status = ac_status_word();
  CUtensorMap map;
  if (!status || !c8_make_map(&map, pages, n_pages, G, ps, d)) return QD_ERR_UNSUPPORTED;
  const AcPlan plan = ac_plan(T, R, H, G, window, max_keys, sms);
  const long long behind = plan.tiles * G - plan.whole, ctas = plan.whole + behind * plan.shares;
  if (ctas > 0x7fffffffll || behind * (AC_ROWS / AC_JOIN_ROWS) > 0x7fffffffll || (behind && !scratch)) return QD_ERR_UNSUPPORTED;
  const AcParams p = {(const bf16*)q, ldq, (bf16*)out, ldo, (const unsigned char*)pages, c8_page_bytes(G, ps, d), (int)n_pages, table, max_blocks, cu,
                      start, R, rows, H, G, ps, ps & (ps - 1) ? -1 : __builtin_ctz(ps), window, AC_ROWS / (H / G), scale * 1.4426950408889634f,
                      (int)plan.tiles, (int)plan.whole, plan.shares, scratch, scratch + behind * plan.shares * AC_ROWS * d, status};
  return d == 64 ? ac_launch<64>(map, p, stream) : ac_launch<128>(map, p, stream);
}

QD_DEFINE_WAIT_PROBE(qd_prefill_attention_fp8_wait_probe, tc_wait(bar, 0, dead, 0, poll_limit), ac_status_word, 99)

// 0 if no kernel of this library has recorded a wait that ran out on the current device.  Synchronises.
extern "C" int qd_prefill_attention_fp8_status() {
  int* status = ac_status_word();
  if (!status) return -1;
  int v = 0;
  if (cudaMemcpy(&v, status, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) return -1;
  if (v) cudaMemset(status, 0, sizeof(int));
  return v;
}
