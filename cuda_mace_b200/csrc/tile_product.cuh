// Products of 16-bit operands on tcgen05 (kind::f16, float32 accumulator in tensor memory) with the epilogues that the dense
// operators need: the gated feed-forward block (gated_feed_forward.cu) and the Newton-Schulz products (orthogonalize.cu).
//
//   D[i, j] = sum over segments, k of A_s[i, k] B_s[k, j]
//
// Operands are read where they lie, row-major with rows of a multiple of 16 bytes: the contracted index may be the inner one
// (K-major) or the outer one (MN-major), so neither a weight nor an activation is ever transposed.  TMA brings tiles of 64 k
// into a ring of stages (128-byte swizzle, zeros outside the array, which is all that ragged sizes need).
//
// Two precisions:
//  * 16-bit operands (bf16, or fp16 where the caller knows the range): one MMA a k step, the sum stays in tensor memory for
//    the whole of K.
//  * PAIR: float32 values as two fp16 values, x = (hi + lo) / scale, hi and lo rounded to nearest: at most 2^-22 |x| off, about 2^-24
//    on the average.  Three MMAs a k step (lo hi, hi lo, hi hi; lo lo is below 2^-22 of hi hi).  fp16 lacks float32's range, so
//    every block of 64 x 64 values has a power of two of its own, from the block's largest value, and lo is kept times 2^11: the terms that it
//    is in are summed first and the first hi hi adds 2^-11 of them.  Within a block the precision holds over 2^28 below that value
//    and degrades to an absolute 2^-50 of it beyond (rows of a caller's array are brought to one size first, row_size).  A block of 64 k is one chunk: its sum goes
//    to its own accumulator columns and the epilogue warps add it, times the two blocks' scales, to float32 registers, rounding to
//    nearest.  That also keeps the tensor core's own accumulation, which truncates, to the four instructions of hi hi: summed in tensor
//    memory over K = 512, three terms of it are off by 4e-6 of the largest value; in chunks all sums come out smaller by 0.9e-7 (terms of
//    either sign) to 1.5e-7 (of one), which the scale that they are multiplied with anyway puts back: 1 + 2^-23.  (Twelve
//    instructions, the terms in turn: 2.0e-7 to 2.9e-7, 1 + 2^-22.)
//    Compared with TF32 in three terms the operands are half as large and the instructions twice as fast.
//
// One persistent CTA an SM, 19 warps: 16 for the epilogue (four a quarter of the 128 tensor-memory lanes, each a quarter of
// the columns; with eight, two a scheduler, they waited for each other's barriers, copies and special functions most of the time), one
// thread that issues the copies, one that issues the MMAs, and a warp that fetches the blocks' scales ahead (the epilogue warps waited
// 700 cycles a segment for them: 47 of the 180 us of the backward's hidden values at 64 000 rows, widths 128 and 512).  Two to four sets of accumulator
// columns: the products of the next chunks or tiles run while the epilogue reads this one's.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstring>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace cmace {

constexpr int TP_EPILOGUE_WARPS = 16;
constexpr int TP_THREADS = (TP_EPILOGUE_WARPS + 3) * 32;   // 96 registers a thread: 64 sums of a PAIR tile and their handling
constexpr int TP_SMEM_BUDGET = 227 * 1024 - 1024;          // without the static barriers
constexpr int TP_MAX_STAGES = 8;

// GATED: D = act(x Wg) * (x Wu).  BACK: what the block's backward needs of a hidden value: h, and the gradients of both
// projections.  GRAM, POLY, APPLY: the three products of a Newton-Schulz step.
enum TpKind { TP_PLAIN, TP_GATED, TP_BACK, TP_GRAM, TP_POLY, TP_APPLY };
enum TpAct { TP_SILU = 0, TP_GELU = 1 };

struct TpOperand {
  CUtensorMap map;         // [z][rows][columns] in boxes of 64 x 64: one map whichever index is contracted
  const float *scale;      // PAIR: inverse scales of the blocks (1 / scale), null where there are none
  int64_t sc_i, sc_k, sc_b;  // their strides over blocks of the free index, of k, and over batches
  int mn_major;            // the contracted index is the outer one
  int z0, zstep;           // hi (or the values) of batch b is matrix z0 + b zstep, lo the one behind it
};

struct TpOut {
  CUtensorMap map;         // boxes of 32 rows
  void *ptr;               // rows that TMA cannot address (not a multiple of 16 bytes): stored by the warps
  int64_t ld, batch;       // elements a row and a batch, for ptr
  int use_map;
};

// Division of u < 2^31 by a number that the host knows (Granlund and Montgomery).  Every role finds its tiles by itself, and one thread issues
// the MMAs: with divisions there, two thirds of the instructions of a short tile were these.
struct TpDiv {
  uint32_t mul, shift;
};
inline TpDiv tp_div(uint32_t d) {
  uint32_t shift = 0;
  while (((uint64_t)1 << shift) < d) shift++;
  return {(uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1), shift};
}
__device__ __forceinline__ uint32_t operator/(uint32_t u, const TpDiv &d) { return (__umulhi(d.mul, u) + u) >> d.shift; }

struct TpArgs {
  TpOperand a[2], b[3];
  TpOut out[2];                  // 16-bit values, hi and lo; results
  float *out_scale[3];           // PAIR outputs with block scales: inverse scale of every 64 x 64 block
  int64_t out_scale_ld, out_scale_batch;
  CUtensorMap cin;               // POLY: S, APPLY: X, in boxes of 32 rows of a warp's columns; batch b is hi 2 b and lo 2 b + 1
  float alpha, beta, pair_scale;   // D = alpha * product + beta * cin, times pair_scale where D is a pair
  const float4 *own;               // Newton-Schulz: a batch's own (a, b, c, ss), (sp, out, ..) of the step, own_stride apart; ss = 0: the three above
  int own_stride;
  const float *row_size[2];        // PAIR: powers of two that A's rows were brought to one size by, [rows up to a multiple of 256]; PLAIN: null: none
  int32_t *status;
  int64_t rows, cols;            // of the output
  int kblocks[2], segments;      // blocks of 64 k a segment
  int last16[2];                 // steps of 16 k in the last of them
  int batches, splits, mt, nt;
  TpDiv by_nt, by_mt, by_batches, by_splits;
  int64_t total;                 // tiles
  int a_of_last;                 // the last batch takes a[1] (its own, unbatched operand) in place of a[0]
  int out_of_batch;              // PLAIN: batch b goes to out[b], an array of its own
  int out_bf16;                  // PLAIN, APPLY's result: 16-bit output
  int in_f16;                    // 16-bit operands are fp16, not bf16
};

__device__ __forceinline__ void umma_16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D = A B + D 2^-11
__device__ __forceinline__ void umma_16_low(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p, 11;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc)
      : "memory");
}
__device__ __forceinline__ void umma_16_low_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p, 11;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc)
      : "memory");
}
__device__ __forceinline__ void umma_16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// a pair's copies count on the first CTA's barrier, its products on both CTAs' (the same place in each)
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"((uint16_t)3)
               : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// One thread of every CTA of a cluster arrives on the barrier of each other, for its block (which has met at bar.sync before), and all threads
// wait on their own CTA's: some 700 cycles where barrier.cluster of 512 threads takes 2 000.
__device__ __forceinline__ void peer_arrive(uint32_t bar, uint32_t rank) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(peer_smem(bar, rank)) : "memory");
}
__device__ __forceinline__ bool peer_wait(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if (clock64() - t0 > GT_TIMEOUT_CYCLES) return false;
  }
}
// Before a CTA's shared memory is written by others of its cluster, they have to know that it runs: arrived on at the start, waited for late.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Says that tensor memory has been read, which tcgen05.fence orders: a release here would wait for all of the warp's stores.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Operand image of rows of 128 bytes with the 128-byte swizzle.  K-major: a row is 64 k of one i, groups of eight rows 1 024 bytes
// apart.  MN-major: a row is 64 i of one k, groups of eight k 1 024 bytes apart (stride offset), runs of 64 i 8 192 (leading offset).
__device__ __forceinline__ uint64_t tp_desc(uint32_t smem, int mn_major) {
  return (uint64_t)((smem & 0x3FFFF) >> 4) | ((uint64_t)(mn_major ? 512 : 1) << 16) | ((uint64_t)64 << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
// kind::f16: D float32, A and B fp16 (0) or bf16 (1) at bits 7 and 10, MN-major operands at bits 15 and 16
__device__ __forceinline__ uint32_t tp_idesc(int n, int bf16, int a_mn, int b_mn, int m = 128) {
  return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// TN: output columns of a tile.  CTAS = 2: a pair of CTAs works on one tile of 256 rows, each with its 128 rows of A and of the sum and
// with half of B's columns in its shared memory, which the pair's MMAs read from both.
template <int KIND, bool PAIR, int TN, int CTAS>
struct TpShape {
  // columns of B a segment: both projections' side by side; BACK's second segment has one's
  static constexpr int N0 = KIND == TP_GATED || KIND == TP_BACK ? 2 * TN : TN, N1 = KIND == TP_BACK ? TN : N0;
  static constexpr int B_ROWS = N0 / CTAS;                  // of a stage of a CTA
  static constexpr int A_BYTES = 128 * 128, B_BYTES = B_ROWS * 128;
  static constexpr int STAGE = (A_BYTES + B_BYTES) * (PAIR ? 2 : 1);
  // BACK's sums of 128 columns do not fit twice: the second segment goes first, into columns that alternate, and the first waits
  // for the epilogue of the tile before.
  static constexpr bool LATE = KIND == TP_BACK && !PAIR && TN == 128;
  // sets of accumulator columns, of a chunk (PAIR) or a tile; LATE: of the second segment
  static constexpr int ACC_COLS = KIND == TP_BACK && !PAIR ? N0 + N1 : N0;
  static constexpr int BUFFERS = LATE ? 2 : (ACC_COLS <= 128 ? 4 : 2), BUFFER_COLS = 512 / BUFFERS;
  static_assert(LATE || ACC_COLS <= BUFFER_COLS, "accumulators");
  static constexpr int PART = TN / 4, EACH = PART / 16;   // a warp's columns of a sum, and in groups of 16
  // Bytes an epilogue warp stages its output in.  A piece is 32 rows of 64 bytes: 16 float32 or 32 16-bit columns; 16 of those are half a
  // piece.  BACK of 16-bit operands: three arrays at once.  Newton-Schulz: hi and lo of a warp's 32 x PART values,
  // GRAM, where nothing comes in, one after the other.
  static constexpr int STAGING = KIND >= TP_GRAM ? (KIND == TP_GRAM ? 1 : 2) * 32 * PART * 2 : (KIND == TP_BACK && !PAIR ? 3 * 1024 : 2048);
  static constexpr int FIT = (TP_SMEM_BUDGET - 1024 - TP_EPILOGUE_WARPS * STAGING) / STAGE;
  static constexpr int STAGES = FIT < TP_MAX_STAGES ? FIT : TP_MAX_STAGES;
  static constexpr int SMEM = STAGE * STAGES + TP_EPILOGUE_WARPS * STAGING + 1024;
};

struct TpTile {
  int64_t row0;
  int n0, batch, split;
};
__device__ __forceinline__ TpTile tp_tile(const TpArgs &g, int64_t t, int out_n, int out_m) {
  TpTile T;
  const uint32_t u = (uint32_t)t, v = u / g.by_nt, w = v / g.by_mt;
  T.n0 = (int)(u - v * (uint32_t)g.nt) * out_n;
  T.row0 = (int64_t)(v - w * (uint32_t)g.mt) * out_m;
  T.split = (int)(w / g.by_batches);
  T.batch = (int)(w - (uint32_t)T.split * (uint32_t)g.batches);
  return T;
}
// k blocks of a split (fewer than 2^25 of them, 64 splits at most)
__device__ __forceinline__ void tp_range(const TpArgs &g, int split, int seg, int &k0, int &k1) {
  const uint32_t n = (uint32_t)g.kblocks[seg];
  k0 = (int)(n * (uint32_t)split / g.by_splits);
  k1 = (int)(n * (uint32_t)(split + 1) / g.by_splits);
}

__device__ __forceinline__ void tp_report(const TpArgs &g, int code) {
  if (g.status) atomicCAS(g.status, 0, code);
}
// named barrier of a part of the epilogue warps
__device__ __forceinline__ void tp_bar(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// power of two that brings `most` (finite, >= 0) into [2^14, 2^15)
__device__ __forceinline__ float tp_scale(float most) {
  int k = 14 - (int)((__float_as_uint(most) >> 23) - 127);   // a subnormal counts as 2^-127
  if (most == 0.f) k = 0;
  k = k > 126 ? 126 : k;
  return __uint_as_float((uint32_t)(k + 127) << 23);
}
__device__ __forceinline__ float tp_finite_abs(float x) {
  const float a = fabsf(x);
  return a < CUDART_INF_F ? a : 0.f;   // infinities and NaN do not set a block's scale
}
// Largest finite magnitude of a thread's values.  Without an infinity that is a maximum with the sign left out, which drops NaN by
// itself: one instruction a value.
template <int N>
__device__ __forceinline__ float tp_most(const float (&v)[N], float most = 0.f) {
#pragma unroll
  for (int j = 0; j < N; j++) most = fmaxf(most, fabsf(v[j]));
  if (most < CUDART_INF_F) return most;
  most = 0.f;
#pragma unroll 1
  for (int j = 0; j < N; j++) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < N; k++) x = k == j ? v[k] : x;
    most = fmaxf(most, tp_finite_abs(x));
  }
  return most;
}
// Two values times a power of two as (hi, lo) pairs of fp16, lo times 2^11.  What is not finite has NaN for lo, and products with it come out NaN.
__device__ __forceinline__ void tp_split2(float x, float y, float scale, uint32_t &hi, uint32_t &lo) {
  const unsigned long long v = mul2(pack2(x, y), pack2(scale, scale));
  float a, b;
  unpack2(v, a, b);
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  unpack2(mul2(sub2(v, pack2(f.x, f.y)), pack2(0x1p11f, 0x1p11f)), a, b);
  const __half2 l = __floats2half2_rn(a, b);
  hi = *reinterpret_cast<const uint32_t *>(&h);
  lo = *reinterpret_cast<const uint32_t *>(&l);
}
// sums += scale * 16 accumulator columns
__device__ __forceinline__ void tp_add(float (&sum)[16], const uint32_t (&v)[16], float scale) {
  const unsigned long long s2 = pack2(scale, scale);
#pragma unroll
  for (int j = 0; j < 16; j += 2)
    unpack2(fma2(pack2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), s2, pack2(sum[j], sum[j + 1])), sum[j], sum[j + 1]);
}
__device__ __forceinline__ uint32_t tp_bf16x2(float x, float y) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t tp_f16x2(float x, float y) {
  const __half2 v = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// Special-function unit without the library functions' care for subnormal results, which are zeros here: two ulp each
__device__ __forceinline__ float tp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// of x times a power of two, which goes into the constant
__device__ __forceinline__ float tp_sigmoid(float x, float size) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + tp_ex2(-1.4426950408889634f * size * x)));
  return y;
}
// Cumulative normal distribution of x = g size.  Its tail is erfc(z) / 2 with z = |x| / sqrt 2, and erfc(z) = e^(-z^2) W(z) with a smooth W that goes
// as 1 / z: a polynomial of t = 1 / (1 + 0.37 z), fitted to W's relative error over 1 + z^2 (which is how the exponential's grows) by least squares
// that were weighted again until the largest was least: 2e-7 of it, 6e-7 in float32 around zero, 1.8e-6 at z = 3.  So the tail keeps its
// precision far below zero, without a branch (erff has two ways, which the lanes of a warp both go).  e: e^(-x^2 / 2), which the derivative takes as well.
__device__ __forceinline__ float tp_normal_cdf(float g, float size, float &e) {
  const float p = g * (0.84932180028801904f * size);   // e^(-x^2 / 2) = 2^(-p^2)
  float t;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.30804531f, fabsf(p), 1.0f)));
  e = tp_ex2(-p * p);
  float w = -0.07034614f;   // half of W
  constexpr float C[] = {0.21358304f, -0.08555056f, 0.15171303f, 0.07971248f, 0.10662103f, 0.10426704f};
#pragma unroll
  for (int k = 0; k < 6; k++) w = fmaf(t, w, C[k]);
  const float tail = t * w * e;
  return g < 0.f ? tail : 1.0f - tail;   // NaN stays NaN
}
// act(x) / x of x = g size, size a power of two; with act'(x)
template <int ACT>
__device__ __forceinline__ float tp_gate(float g, float size) {
  if (ACT == TP_SILU) return tp_sigmoid(g, size);
  float e;
  return tp_normal_cdf(g, size, e);
}
template <int ACT>
__device__ __forceinline__ float tp_gate(float g, float size, float &d) {
  if (ACT == TP_SILU) {
    const float s = tp_sigmoid(g, size);
    d = s * fmaf(size, g - g * s, 1.0f);
    return s;
  }
  float e;
  const float cdf = tp_normal_cdf(g, size, e);
  d = cdf + 0.39894228040143268f * size * g * e;
  return cdf;
}
template <int ACT>
__device__ __forceinline__ float tp_act(float g) { return g * tp_gate<ACT>(g, 1.f); }

// ---- an epilogue warp's stores ------------------------------------------------------------------------------------------
struct TpStager {
  uint32_t smem;
  int lane;
  int64_t rows, cols;   // of the output: a box that starts outside is not stored
  __device__ __forceinline__ void begin() const {   // the copy engine has read what was staged before
    if (elect_one()) tma_store_wait_read();
    __syncwarp();
  }
  // 16-byte chunks chunk, chunk + 1, ... of this lane's row of a piece at `at` (rows of 64 bytes) or half a piece (32 bytes)
  template <int ROW_BYTES>
  __device__ __forceinline__ uint4 get(uint32_t at, int chunk) const {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem + at + offset<ROW_BYTES>(lane, chunk)) : "memory");
    return v;
  }
  template <int ROW_BYTES, int WORDS>
  __device__ __forceinline__ void put(uint32_t at, int chunk, const uint32_t (&w)[WORDS]) const {
#pragma unroll
    for (int c = 0; c < WORDS / 4; c++)
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem + at + offset<ROW_BYTES>(lane, chunk + c)), "r"(w[4 * c]),
                   "r"(w[4 * c + 1]), "r"(w[4 * c + 2]), "r"(w[4 * c + 3])
                   : "memory");
  }
  // the copy engine's swizzles of rows of 128, 64 and 32 bytes
  template <int ROW_BYTES>
  static __device__ __forceinline__ uint32_t offset(int row, int chunk) {
    return ROW_BYTES == 128 ? (uint32_t)sw128_offset(row, chunk) : ROW_BYTES == 64 ? (uint32_t)sw64_offset(row, chunk) : (uint32_t)(row * 32 + ((chunk ^ ((row >> 2) & 1)) << 4));
  }
  __device__ __forceinline__ void send(const CUtensorMap *map, uint32_t at, int col, int64_t row, int batch) const {
    fence_proxy_async();
    __syncwarp();
    if (row < rows && col < cols && elect_one()) tma_store_3d(map, col, (int)row, batch, smem + at);
  }
  // rows that TMA cannot address, from a piece: two rows an instruction, a lane has one float32 or two 16-bit columns
  __device__ __forceinline__ void send_rows(const TpOut &o, bool sixteen, uint32_t piece, int col, int64_t row, int batch) const {
    __syncwarp();
    const int w = lane & 15, r0 = lane >> 4, n = (int)(rows - row < 32 ? rows - row : 32);
    uint32_t v[16];
#pragma unroll
    for (int i = 0; i < 16; i++)
      asm volatile("ld.shared.b32 %0, [%1];"
                   : "=r"(v[i])
                   : "r"(smem + piece + (uint32_t)sw64_offset(r0 + 2 * i, w >> 2) + 4u * (uint32_t)(w & 3))
                   : "memory");
    const int64_t at = (int64_t)batch * o.batch + (row + r0) * o.ld + col + (sixteen ? 2 * w : w);
    if (!sixteen) {
      uint32_t *p = static_cast<uint32_t *>(o.ptr) + at;
#pragma unroll
      for (int i = 0; i < 16; i++, p += 2 * o.ld)
        if (r0 + 2 * i < n && col + w < cols) *p = v[i];
    } else {
      uint16_t *p = static_cast<uint16_t *>(o.ptr) + at;
#pragma unroll
      for (int i = 0; i < 16; i++, p += 2 * o.ld) {
        if (r0 + 2 * i < n && col + 2 * w < cols) p[0] = (uint16_t)v[i];
        if (r0 + 2 * i < n && col + 2 * w + 1 < cols) p[1] = (uint16_t)(v[i] >> 16);
      }
    }
    __syncwarp();
  }
};

template <int KIND, bool PAIR, int TN, int CTAS, int ACT>
__global__ void __launch_bounds__(TP_THREADS, 1) tile_product_kernel(const __grid_constant__ TpArgs g) {
  using S = TpShape<KIND, PAIR, TN, CTAS>;
  constexpr int TERMS = PAIR ? 2 : 1;
  constexpr int STAGES = S::STAGES, ROWS = 128 * CTAS;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * TP_MAX_STAGES + 13 + TP_EPILOGUE_WARPS];
  __shared__ uint32_t tmem_base_slot;
  __shared__ float block_most[2][3][TP_EPILOGUE_WARPS];   // of alternating tiles, of BACK's three outputs
  __shared__ float scales[4][8];   // of the chunk in each set of columns: products of the inverse scales, [block of rows][of columns][projection]
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t staging = smem + (uint32_t)(STAGES * S::STAGE);
  const uint32_t full = smem_u32(&bars[0]), empty = smem_u32(&bars[TP_MAX_STAGES]);
  const uint32_t acc_full = smem_u32(&bars[2 * TP_MAX_STAGES]), acc_empty = smem_u32(&bars[2 * TP_MAX_STAGES + 4]);
  const uint32_t drain = smem_u32(&bars[2 * TP_MAX_STAGES + 8]);
  const uint32_t scale_empty = drain + 8 + 8 * TP_EPILOGUE_WARPS;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = CTAS == 2 ? (int)cluster_rank() : 0;
  const int64_t first_tile = blockIdx.x / CTAS, tile_step = gridDim.x / CTAS;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(full + 8 * s, 1);    // the copies' expect_tx
      mbar_init(empty + 8 * s, 1);   // one commit
    }
    for (int b = 0; b < S::BUFFERS; b++) {
      mbar_init(acc_full + 8 * b, PAIR ? 2 : 1);                // one commit, the scales' arrival
      mbar_init(acc_empty + 8 * b, CTAS * TP_EPILOGUE_WARPS);   // one arrival a warp
    }
    mbar_init(drain, 1);
    for (int b = 0; b < S::BUFFERS; b++) mbar_init(scale_empty + 8 * b, TP_EPILOGUE_WARPS);
    for (int w = 0; w < TP_EPILOGUE_WARPS; w++) mbar_init(drain + 8 + 8 * w, 1);   // a warp's own copies
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == TP_EPILOGUE_WARPS) {
    if (CTAS == 2) tmem_alloc_pair(smem_u32(&tmem_base_slot), 512);
    else tmem_alloc(smem_u32(&tmem_base_slot), 512);
  }
  tc_fence_before();
  __syncwarp();
  if (CTAS == 2) cluster_sync();   // the other CTA's barriers
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)uniform((int)tmem_base_slot);
  if (threadIdx.x < 5) {   // the maps are arguments: fetched before the wait
    const CUtensorMap *map = threadIdx.x < 2 ? &g.a[threadIdx.x].map : &g.b[threadIdx.x - 2].map;
    if (threadIdx.x == 0 || threadIdx.x == 2 || (threadIdx.x == 4 ? KIND == TP_BACK : g.segments > 1 || KIND == TP_GATED || KIND == TP_BACK || g.a_of_last))
      asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }
  grid_wait();
  grid_release();   // after the allocation

  if (warp == TP_EPILOGUE_WARPS) {
    // ================================ copies ================================
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0, used = 0;   // used: bit per stage that has been filled at least once
      bool ok = true;
      const uint32_t first_full = CTAS == 2 ? peer_smem(full, 0) : full;
      for (int64_t t = first_tile; ok && t < g.total; t += tile_step) {
        const TpTile T = tp_tile(g, t, TN, ROWS);
        for (int i = 0; ok && i < g.segments; i++) {
          const int seg = S::LATE ? 1 - i : i;
          const bool last = g.a_of_last && T.batch == g.batches - 1;
          const TpOperand &A = g.a[last ? 1 : seg];
          int k0, k1;
          tp_range(g, T.split, seg, k0, k1);
          const int rows = (seg == 0 ? S::N0 : S::N1) / CTAS;   // of B; 32 are copied as 64
          const int boxes = (rows + 63) / 64;
          const uint32_t bytes = (uint32_t)(CTAS * TERMS * (S::A_BYTES + boxes * 8192));
          const int row0 = (int)T.row0 + 128 * rank;
          for (int kb = k0; kb < k1; kb++) {
            if (!mbar_wait(empty + 8 * stage, phase ^ 1)) {
              tp_report(g, 100);
              ok = false;
              break;
            }
            const uint32_t bar = first_full + 8 * stage, sA = smem + (uint32_t)(stage * S::STAGE);
            const uint32_t sB = sA + TERMS * S::A_BYTES;
            const int k = kb * 64;
            if (rank == 0) mbar_arrive_expect_tx(full + 8 * stage, bytes);
            // a box is 64 rows of 128 bytes, of the free index (K-major) or of k (MN-major)
            const auto copy = [&](const TpOperand &o, uint32_t to, int at, int term) {
              const int x = o.mn_major ? at : k, y = o.mn_major ? k : at, z = o.z0 + T.batch * o.zstep + term;
              if (CTAS == 2) tma_load_3d_pair(to, &o.map, x, y, z, bar);
              else tma_load_3d(to, &o.map, x, y, z, bar);
            };
#pragma unroll
            for (int term = 0; term < TERMS; term++) {
              copy(A, sA + term * S::A_BYTES, row0, term);
              copy(A, sA + term * S::A_BYTES + 8192, row0 + 64, term);
              for (int b = 0; b < boxes; b++) {
                const int n = rank * rows + 64 * b;   // column of the segment's B
                int which = seg, at = n;
                if (KIND == TP_GATED || KIND == TP_BACK) {
                  which = seg == 1 ? 2 : n / TN;
                  at = seg == 1 ? n : n - which * TN;
                }
                copy(g.b[which], sB + term * S::B_BYTES + (uint32_t)(8192 * b), T.n0 + at, term);
              }
            }
            used |= 1u << stage;
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1;
            }
            // What the first tile's epilogue adds comes behind the first operands: in front of them it kept the products waiting for up to 7 us.
            if constexpr (KIND == TP_POLY || KIND == TP_APPLY) {
              if (t == first_tile && kb + 1 == (k1 - k0 < STAGES ? k1 : k0 + STAGES)) {
                for (int w = 0; w < TP_EPILOGUE_WARPS; w++) {
                  const int row = row0 + 32 * (w & 3), col = T.n0 + (w >> 2) * S::PART;
                  if (row >= g.rows || col >= g.cols) continue;
                  const uint32_t to = staging + (uint32_t)(w * S::STAGING), cin_bar = drain + 8 + 8 * (uint32_t)w;
                  mbar_arrive_expect_tx(cin_bar, 2 * 32 * S::PART * 2);
                  tma_load_3d(to, &g.cin, col, row, 2 * T.batch, cin_bar);
                  tma_load_3d(to + 32 * S::PART * 2, &g.cin, col, row, 2 * T.batch + 1, cin_bar);
                }
              }
            }
          }
        }
      }
      if (!ok && rank == 0) {   // no copy outlives the block: the fills that nobody took
        for (int s = 0; s < STAGES; s++)
          if (used >> s & 1) mbar_wait(full + 8 * s, s < stage ? phase : phase ^ 1);
      }
    }
  } else if (warp == TP_EPILOGUE_WARPS + 1) {
    // ================================ products ================================
    if (rank == 0 && elect_one()) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, uses = 0;   // uses: bit per set of columns, the parity of its uses
      const auto next_buffer = [&] {
        uses ^= 1u << buf;
        buf = buf + 1 == S::BUFFERS ? 0 : buf + 1;
      };
      bool ok = true;
      const int bf16 = g.in_f16 || PAIR ? 0 : 1;
      const auto product = [&](uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
        if (CTAS == 2) umma_16_pair(d, a, b, idesc, accumulate);
        else umma_16(d, a, b, idesc, accumulate);
      };
      const auto commit = [&](uint32_t bar) {
        if (CTAS == 2) umma_commit_pair(bar);
        else umma_commit(bar);
      };
      for (int64_t t = first_tile; ok && t < g.total; t += tile_step) {
        const TpTile T = tp_tile(g, t, TN, ROWS);
        if (!PAIR) {
          if (!mbar_wait(acc_empty + 8 * buf, (uses >> buf & 1) ^ 1)) {
            tp_report(g, 101);
            break;
          }
          tc_fence_after();
        }
        uint32_t begun = 0;
        for (int i = 0; ok && i < g.segments; i++) {
          const int seg = S::LATE ? 1 - i : i;
          int k0, k1;
          tp_range(g, T.split, seg, k0, k1);
          const bool last = g.a_of_last && T.batch == g.batches - 1;
          const int a_mn = g.a[last ? 1 : seg].mn_major;
          const int b_mn = g.b[KIND == TP_BACK ? 2 * seg : (KIND == TP_GATED ? 0 : seg)].mn_major;
          const uint32_t idesc = tp_idesc(seg == 0 ? S::N0 : S::N1, bf16, a_mn, b_mn, ROWS);
          const uint64_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;   // 16 k, in units of 16 bytes
          if (KIND == TP_BACK) begun = 0;
          if (S::LATE && seg == 0 && !mbar_wait(acc_empty + 8 * (buf ^ 1), (uses >> (buf ^ 1) & 1) ^ 1)) {
            tp_report(g, 108);
            ok = false;
            break;
          }
          if (S::LATE) tc_fence_after();
          for (int kb = k0; kb < k1; kb++) {
            if (PAIR) {
              if (!mbar_wait(acc_empty + 8 * buf, (uses >> buf & 1) ^ 1)) {
                tp_report(g, 102);
                ok = false;
                break;
              }
            }
            if (!mbar_wait(full + 8 * stage, phase)) {
              tp_report(g, 103);
              ok = false;
              break;
            }
            tc_fence_after();
            uint32_t d = tmem + (uint32_t)(buf * S::BUFFER_COLS);
            if (KIND == TP_BACK && !PAIR) d = S::LATE ? tmem + (seg == 0 ? 0u : 256u + 128u * (uint32_t)buf) : d + (seg == 0 ? 0u : 2u * TN);
            const uint32_t sA = smem + (uint32_t)(stage * S::STAGE), sB = sA + TERMS * S::A_BYTES;
            const uint64_t a_hi = tp_desc(sA, a_mn), b_hi = tp_desc(sB, b_mn);
            if (PAIR) {   // low parts first: what they sum to is 2^11 times itself
              const uint64_t a_lo = tp_desc(sA + S::A_BYTES, a_mn), b_lo = tp_desc(sB + S::B_BYTES, b_mn);
#pragma unroll
              for (int ks = 0; ks < 4; ks++) {
                product(d, a_lo + ks * a_step, b_hi + ks * b_step, idesc, ks > 0);
                product(d, a_hi + ks * a_step, b_lo + ks * b_step, idesc, 1);
              }
              if (CTAS == 2) umma_16_low_pair(d, a_hi, b_hi, idesc);
              else umma_16_low(d, a_hi, b_hi, idesc);
#pragma unroll
              for (int ks = 1; ks < 4; ks++) product(d, a_hi + ks * a_step, b_hi + ks * b_step, idesc, 1);
            }
#pragma unroll
            for (int ks = 0; ks < (PAIR ? 0 : 4); ks++) {
              product(d, a_hi + ks * a_step, b_hi + ks * b_step, idesc, begun);
              begun = 1;
            }
            commit(empty + 8 * stage);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1;
            }
            if (PAIR) {
              commit(acc_full + 8 * buf);
              next_buffer();
            }
          }
        }
        if (!PAIR && ok) {
          commit(acc_full + 8 * buf);
          next_buffer();
        }
      }
      commit(drain);   // nothing of this block's products is in flight when the columns are given back
      if (!mbar_wait(drain, 0)) tp_report(g, 104);
    }
  } else if (warp == TP_EPILOGUE_WARPS + 2) {
    // ================================ scales ================================
    // four chunks at a time, eight lanes each
    if (PAIR) {
      uint32_t chunk = 0;   // of this block
      bool ok = true;
      const int block_row = (lane >> 2) & 1, block_col = (lane >> 1) & 1, projection = lane & 1;
      constexpr bool TWO = KIND == TP_GATED || KIND == TP_BACK;   // both projections in the first segment
      for (int64_t t = first_tile; ok && t < g.total; t += tile_step) {
        const TpTile T = tp_tile(g, t, TN, ROWS);
        const int64_t row = T.row0 + 128 * rank + 64 * block_row;
        const int col = T.n0 + (TN == 64 ? 0 : 64 * block_col);
        for (int seg = 0; ok && seg < g.segments; seg++) {
          const bool last = g.a_of_last && T.batch == g.batches - 1;
          const TpOperand &A = g.a[last ? 1 : seg], &B = g.b[TWO ? (seg == 0 ? projection : 2) : seg];
          int k0, k1;
          tp_range(g, T.split, seg, k0, k1);
          // past the end there are zeros, in any scale
          const float *pa = A.scale && row < g.rows ? A.scale + T.batch * A.sc_b + (row >> 6) * A.sc_i : nullptr;
          const float *pb = B.scale && col < g.cols ? B.scale + T.batch * B.sc_b + (col >> 6) * B.sc_i : nullptr;
          for (int kb = k0; ok && kb < k1; kb += 4) {
            const int mine = kb + (lane >> 3), n = k1 - kb < 4 ? k1 - kb : 4;
            // what truncation takes, by the additions that have something to add
            const int steps = mine + 1 == g.kblocks[seg] ? g.last16[seg] : 4;
            float a = steps > 2 ? 1.f + 0x1p-23f : 1.f, b = 1.f;
            if (mine < k1) {
              if (pa) a *= __ldcg(pa + mine * A.sc_k);
              if (pb) b = __ldcg(pb + mine * B.sc_k);
            }
            for (int i = 0; ok && i < n; i++, chunk++) {
              const uint32_t set = chunk % S::BUFFERS;
              if (!warp_wait(scale_empty + 8 * set, (chunk / S::BUFFERS & 1) ^ 1, lane)) {
                if (lane == 0) tp_report(g, 111);
                ok = false;
                break;
              }
              if (lane >> 3 == i) scales[set][lane & 7] = a * b;
              __syncwarp();
              if (lane == 0) mbar_arrive(acc_full + 8 * set);
            }
          }
        }
      }
    }
  } else {
    // ================================ epilogue ================================
    const int q = warp & 3, part = warp >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    const TpStager st{staging + (uint32_t)(warp * S::STAGING), lane, g.rows, g.cols};
    const uint32_t cin_bar = drain + 8 + 8 * (uint32_t)warp;
    uint32_t cin_phase = 0;
    int buf = 0;
    uint32_t uses = 0;
    const auto next_buffer = [&] {
      uses ^= 1u << buf;
      buf = buf + 1 == S::BUFFERS ? 0 : buf + 1;
    };
    bool ok = true;
    // groups of 16 columns of the sums that this warp owns
    constexpr int EACH = S::EACH;
    constexpr int GROUPS = KIND == TP_BACK ? 3 * EACH : (KIND == TP_GATED ? 2 * EACH : EACH);
    constexpr int SEG0_GROUPS = KIND == TP_BACK ? 2 * EACH : GROUPS;
    static_assert(KIND != TP_GATED || TN == 128, "32 columns of both projections a warp");
    static_assert(!PAIR || TN <= 128, "a warp's columns are of one block of 64");
    const uint32_t first_empty = CTAS == 2 ? peer_smem(acc_empty, 0) : acc_empty;
    const auto release = [&](int b) {   // this warp has read the sums
      tc_fence_before();
      __syncwarp();
      if (ok && lane == 0) {
        if (CTAS == 2) mbar_arrive_cluster(first_empty + 8 * b);
        else mbar_arrive(acc_empty + 8 * b);
      }
    };
    // first column of group i inside the accumulator (BACK: the last sum has an accumulator, or columns, of its own)
    const auto column = [&](int i) -> uint32_t {
      const uint32_t in = (uint32_t)(part * S::PART + 16 * (i % EACH));
      if (KIND == TP_GATED) return (uint32_t)(i / EACH * TN) + in;
      if (KIND == TP_BACK) return i < 2 * EACH ? (uint32_t)(i / EACH * TN) + in : (PAIR ? in : (uint32_t)(2 * TN) + in);
      return in;
    };
    // A warp whose wait gave up goes through the rest of its tiles without waiting: others meet it at the named barriers.
    int odd = 0;
    for (int64_t t = first_tile; t < g.total; t += tile_step, odd ^= 1) {
      const TpTile T = tp_tile(g, t, TN, ROWS);
      const int64_t row = T.row0 + 128 * rank + 32 * q;   // first row of this warp
      const int col0 = T.n0 + part * S::PART;             // first column
      // What a Newton-Schulz epilogue adds to the product, S or X: on its way into the pieces that the warp's values leave by, before the sums
      // are there.  (Loads by the lanes, each of its own row, took as long as the products.)
      constexpr bool CIN = KIND == TP_POLY || KIND == TP_APPLY;
      constexpr uint32_t LOW = 32 * S::PART * 2;   // bytes from a warp's hi to its lo
      const bool here = row < g.rows && col0 < g.cols;
      // of this lane's row: known long before the sums are
      float size[2] = {1.f, 1.f};   // PAIR alone has others
      if constexpr (PAIR && (KIND == TP_GATED || KIND == TP_BACK)) {
        size[0] = __ldcg(g.row_size[0] + (uint32_t)row + lane);
      } else if constexpr (PAIR && KIND == TP_PLAIN) {
        if (g.row_size[0]) size[0] = __ldcg(g.row_size[0] + (uint32_t)row + lane), size[1] = __ldcg(g.row_size[1] + (uint32_t)row + lane);
      }
      if (CIN && here && t != first_tile) {   // the first tile's: by the thread that issues the copies
        if (elect_one()) {
          tma_store_wait_read();
          mbar_arrive_expect_tx(cin_bar, 2 * LOW);
          tma_load_3d(st.smem, &g.cin, col0, (int)row, 2 * T.batch, cin_bar);
          tma_load_3d(st.smem + LOW, &g.cin, col0, (int)row, 2 * T.batch + 1, cin_bar);
        }
        __syncwarp();
      }
      float alpha = g.alpha, beta = g.beta, pair_scale = g.pair_scale;
      if constexpr (KIND >= TP_GRAM) {
        const float4 own = __ldcg(g.own + (int64_t)T.batch * g.own_stride), more = __ldcg(g.own + (int64_t)T.batch * g.own_stride + 1);
        if (own.w != 0.f) {
          if (KIND == TP_GRAM) pair_scale = own.w;
          else if (KIND == TP_POLY) alpha = own.z / (own.w * own.w), beta = own.y / own.w, pair_scale = more.x;
          else alpha = more.y / (more.x * 0x1p15f), beta = own.x * more.y * 0x1p-15f;
        }
      }
      float acc[PAIR ? GROUPS : 1][16];
      if (PAIR) {
#pragma unroll
        for (int i = 0; i < (PAIR ? GROUPS : 1); i++)
#pragma unroll
          for (int j = 0; j < 16; j++) acc[i][j] = 0.f;
#pragma unroll
        for (int seg = 0; seg < 2; seg++) {
          if (seg >= g.segments) break;
          const int i0 = KIND == TP_BACK && seg == 1 ? SEG0_GROUPS : 0;
          const int i1 = KIND == TP_BACK && seg == 0 ? SEG0_GROUPS : GROUPS;
          int k0, k1;
          tp_range(g, T.split, seg, k0, k1);
          constexpr bool TWO = KIND == TP_GATED || KIND == TP_BACK;
          for (int kb = k0; kb < k1; kb++) {
            if (ok && !warp_wait_all(acc_full + 8 * buf, uses >> buf & 1, lane)) {
              if (lane == 0) tp_report(g, 105);
              ok = false;
            }
            const float *scale = scales[buf] + 4 * (q >> 1) + 2 * (part >> 1);   // TN = 64: both blocks of columns are the one
            const float s0 = scale[0], s1 = scale[1];
            tc_fence_after();
            const uint32_t at = lanes + (uint32_t)(buf * S::BUFFER_COLS);
#pragma unroll
            for (int i = 0; i < (PAIR ? GROUPS : 1); i++) {
              if (i < i0 || i >= i1) continue;
              uint32_t v[16];
              tmem_ld16_nowait(at + column(i), v);
              tmem_ld_wait();
              tp_add(acc[i], v, TWO && i / EACH == 1 ? s1 : s0);
            }
            release(buf);
            if (ok && lane == 0) mbar_arrive(scale_empty + 8 * buf);   // after the warp has met in release()
            next_buffer();
          }
        }
      } else {
        if (ok && !warp_wait_all(acc_full + 8 * buf, uses >> buf & 1, lane)) {
          if (lane == 0) tp_report(g, 106);
          ok = false;
        }
        tc_fence_after();
      }
      const uint32_t at = lanes + (S::LATE ? 0u : (uint32_t)(buf * S::BUFFER_COLS));
      // group i of the finished sums
      const auto take = [&](int i, float (&v)[16]) {
        if (PAIR) {
#pragma unroll
          for (int j = 0; j < 16; j++) v[j] = KIND == TP_PLAIN ? acc[PAIR ? i : 0][j] * size[0] * size[1] : acc[PAIR ? i : 0][j];
        } else {
          uint32_t u[16];
          tmem_ld16_nowait(at + column(i) + (S::LATE && i >= SEG0_GROUPS ? 128u * (uint32_t)buf : 0u), u);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; j++) v[j] = __uint_as_float(u[j]);
        }
      };

      if constexpr (KIND == TP_GATED) {
        if constexpr (PAIR) {
          float most = 0.f;
#pragma unroll
          for (int i = 0; i < EACH; i++) {
#pragma unroll
            for (int j = 0; j < 16; j++) acc[i][j] = acc[i][j] * tp_gate<ACT>(acc[i][j], size[0]) * acc[PAIR ? EACH + i : 0][j];
            most = tp_most(acc[i], most);
          }
          // a block of 64 x 64 values is two quarters' and two parts' warps'
          most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
          if (lane == 0) block_most[odd][0][warp] = most;
          tp_bar(1 + 2 * (part >> 1) + (q >> 1), 128);
          const float scale = tp_scale(fmaxf(fmaxf(most, block_most[odd][0][warp ^ 1]), fmaxf(block_most[odd][0][warp ^ 4], block_most[odd][0][warp ^ 5])));
          if (lane == 0 && (q & 1) == 0 && (part & 1) == 0 && row < g.rows && col0 < g.cols)
            g.out_scale[0][(row >> 6) * g.out_scale_ld + (col0 >> 6)] = 1.0f / scale;
          uint32_t w[16], lo[16];
#pragma unroll
          for (int j = 0; j < 16; j++) tp_split2(acc[j >> 3][2 * (j & 7)], acc[j >> 3][2 * (j & 7) + 1], scale, w[j], lo[j]);
          st.begin();
          st.put<64>(0, 0, w);
          st.send(&g.out[0].map, 0, col0, row, 0);
          st.begin();
          st.put<64>(0, 0, lo);
          st.send(&g.out[0].map, 0, col0, row, 1);
        } else {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < EACH; i++) {
            float a[16], u[16];
            take(i, a);
            take(EACH + i, u);
#pragma unroll
            for (int j = 0; j < 8; j++) w[8 * i + j] = tp_bf16x2(tp_act<ACT>(a[2 * j]) * u[2 * j], tp_act<ACT>(a[2 * j + 1]) * u[2 * j + 1]);
          }
          st.begin();
          st.put<64>(0, 0, w);
          st.send(&g.out[0].map, 0, col0, row, 0);
        }
      } else if constexpr (KIND == TP_BACK) {
        // h = act(g) u, dL/dg = dL/dh u act'(g), dL/du = dL/dh act(g); PAIR: all of the rows' common size, but for the g of the gate
        static_assert(!PAIR || TN == 64, "a block of 64 columns a tile");
#pragma unroll
        for (int e = 0; e < EACH; e++) {
          float a[16], u[16], dh[16];
          take(e, a);
          take(EACH + e, u);
          take(2 * EACH + e, dh);
#pragma unroll
          for (int j = 0; j < 16; j++) {
            float d;
            const float act = a[j] * tp_gate<ACT>(a[j], size[0], d);
            const float h = act * u[j], dg = dh[j] * (u[j] * d), du = dh[j] * act;
            a[j] = h;
            u[j] = dg;
            dh[j] = du;
          }
          float scale[3] = {1.f, 1.f, 1.f};
          if (PAIR) {
            float most[3] = {tp_most(u), tp_most(dh), tp_most(a)};
#pragma unroll
            for (int p = 0; p < 3; p++) {
              most[p] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most[p])));
              if (lane == 0) block_most[odd][p][warp] = most[p];
            }
            tp_bar(1 + (q >> 1), 256);   // 64 rows x 64 columns: two quarters, all parts
#pragma unroll
            for (int p = 0; p < 3; p++) {
              float m = 0.f;
#pragma unroll
              for (int k = 0; k < 4; k++) m = fmaxf(m, fmaxf(block_most[odd][p][(q & 2) + 4 * k], block_most[odd][p][(q & 2) + 1 + 4 * k]));
              scale[p] = tp_scale(m);
              if (lane == 0 && (q & 1) == 0 && part == 0 && row < g.rows && T.n0 < g.cols)
                g.out_scale[p][(row >> 6) * g.out_scale_ld + (T.n0 >> 6)] = 1.0f / scale[p];
            }
          }
#pragma unroll
          for (int p = 0; p < 3; p++) {
            uint32_t w[8], lo[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
              const float x = p == 0 ? u[2 * j] : (p == 1 ? dh[2 * j] : a[2 * j]);
              const float y = p == 0 ? u[2 * j + 1] : (p == 1 ? dh[2 * j + 1] : a[2 * j + 1]);
              if (PAIR) tp_split2(x, y, scale[p], w[j], lo[j]);
              else w[j] = tp_bf16x2(x, y);
            }
            if (PAIR) {
              st.begin();
              st.put<32>(0, 0, w);
              st.put<32>(1024, 0, lo);
              st.send(&g.out[0].map, 0, col0, row, 2 * p);
              st.send(&g.out[0].map, 1024, col0, row, 2 * p + 1);
            } else {
              if (p == 0) st.begin();
              st.put<32>(1024 * p, 0, w);
              st.send(&g.out[0].map, 1024 * p, col0 + 16 * e, row, p);
            }
          }
        }
      } else if constexpr (KIND == TP_PLAIN) {
        const TpOut &out = g.out[g.out_of_batch ? T.batch : 1];
        const int batch = g.out_of_batch ? 0 : T.split * g.batches + T.batch;
        if (g.out_bf16) {
#pragma unroll
          for (int i = 0; i < GROUPS; i += 2) {
            const int col = col0 + 16 * i;
            if (col >= g.cols) break;
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 2; k++) {
              float v[16];
              take(i + k, v);
#pragma unroll
              for (int j = 0; j < 8; j++) w[8 * k + j] = tp_bf16x2(v[2 * j], v[2 * j + 1]);
            }
            st.begin();
            st.put<64>(0, 0, w);
            if (out.use_map) st.send(&out.map, 0, col, row, batch);
            else st.send_rows(out, true, 0, col, row, batch);
          }
        } else {
#pragma unroll
          for (int i = 0; i < GROUPS; i++) {
            const int col = col0 + 16 * i;
            if (col >= g.cols) break;
            float v[16];
            take(i, v);
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; j++) w[j] = __float_as_uint(v[j]);
            st.begin();
            st.put<64>(0, 0, w);
            if (out.use_map) st.send(&out.map, 0, col, row, batch);
            else st.send_rows(out, false, 0, col, row, batch);
          }
        }
      } else {
        // Newton-Schulz: values in float32, then hi and lo at a power of two that the caller has from its bounds
        constexpr int ROW = 2 * S::PART;   // bytes of a row of a piece
        if (CIN && here) {
          if (!warp_wait(cin_bar, cin_phase, lane)) {   // after another wait gave up too: no copy outlives the block
            if (lane == 0) tp_report(g, 109);
            ok = false;
          }
          cin_phase ^= 1;
        }
        const bool result = KIND == TP_APPLY && g.pair_scale == 0.f;
        if (!CIN) st.begin();
        float all[GROUPS][16];   // of the result, which leaves in pieces of another shape
#pragma unroll
        for (int i = 0; i < GROUPS; i++) {
          float (&v)[16] = all[i];
          take(i, v);
          if constexpr (CIN) {
            const uint4 x = st.get<ROW>(0, 2 * i), y = st.get<ROW>(0, 2 * i + 1), xl = st.get<ROW>(LOW, 2 * i), yl = st.get<ROW>(LOW, 2 * i + 1);
            const uint32_t hw[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w}, lw[8] = {xl.x, xl.y, xl.z, xl.w, yl.x, yl.y, yl.z, yl.w};
#pragma unroll
            for (int k = 0; k < 8; k++) {
              const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&hw[k])), e = __half22float2(*reinterpret_cast<const __half2 *>(&lw[k]));
              v[2 * k] = alpha * v[2 * k] + beta * fmaf(e.x, 0x1p-11f, a.x);
              v[2 * k + 1] = alpha * v[2 * k + 1] + beta * fmaf(e.y, 0x1p-11f, a.y);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 16; j++) v[j] *= alpha;
          }
          if (!result) {
            uint32_t w[8], lo[8];
#pragma unroll
            for (int j = 0; j < 8; j++) tp_split2(v[2 * j], v[2 * j + 1], pair_scale, w[j], lo[j]);
            st.put<ROW>(0, 2 * i, w);
            if (CIN) st.put<ROW>(LOW, 2 * i, lo);
            else
#pragma unroll
              for (int j = 0; j < 8; j++) v[j] = __uint_as_float(lo[j]);   // GRAM: kept until hi has left
          }
        }
        if (!result) {
          st.send(&g.out[0].map, 0, col0, row, 2 * T.batch);
          if (!CIN) {
            st.begin();
#pragma unroll
            for (int i = 0; i < GROUPS; i++) {
              uint32_t lo[8];
#pragma unroll
              for (int j = 0; j < 8; j++) lo[j] = __float_as_uint(all[i][j]);
              st.put<ROW>(0, 2 * i, lo);
            }
          }
          st.send(&g.out[0].map, CIN ? LOW : 0u, col0, row, 2 * T.batch + 1);
        } else {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < GROUPS; i++) {
            const int col = col0 + 16 * i;
            if (col >= g.cols) break;
            const float (&v)[16] = all[i];
            if (!g.out_bf16) {
              uint32_t w[16];
#pragma unroll
              for (int j = 0; j < 16; j++) w[j] = __float_as_uint(v[j]);
              st.begin();
              st.put<64>(0, 0, w);
              if (g.out[1].use_map) st.send(&g.out[1].map, 0, col, row, T.batch);
              else st.send_rows(g.out[1], false, 0, col, row, T.batch);
            } else if (g.out[1].use_map) {
              uint32_t w[8];
#pragma unroll
              for (int j = 0; j < 8; j++) w[j] = tp_bf16x2(v[2 * j], v[2 * j + 1]);
              st.begin();
              st.put<32>(0, 0, w);
              st.send(&g.out[1].map, 0, col, row, T.batch);
            } else {
              __nv_bfloat16 *o =
                  static_cast<__nv_bfloat16 *>(g.out[1].ptr) + (int64_t)T.batch * g.out[1].batch + (row + lane) * g.out[1].ld + col;
#pragma unroll
              for (int j = 0; j < 16; j++)
                if (row + lane < g.rows && col + j < g.cols) o[j] = __float2bfloat16_rn(v[j]);
            }
          }
        }
      }
      if (!PAIR) {
        release(buf);
        next_buffer();
      }
    }
    if (elect_one()) tma_store_wait_read();   // the copy engine reads this warp's staging buffer; what it writes, the grid's end waits for
  }
  tc_fence_before();
  if (CTAS == 2) {
    __syncthreads();
    __syncwarp();
    cluster_sync();   // the other CTA's products have read this one's operands, its warps have arrived here
    if (warp == TP_EPILOGUE_WARPS) tmem_dealloc_pair(tmem, 512);
  } else {
    __syncthreads();
    if (warp == TP_EPILOGUE_WARPS) tmem_dealloc(tmem, 512);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
// [batch][rows][cols] of 16-bit or float32 values, rows ld elements apart, as boxes of box_cols x box_rows (gemm_tc.cu)
int encode_tile_map(CUtensorMap *map, const void *base, int bytes, bool bf16, int64_t cols, int64_t rows, int64_t batches, int64_t ld,
                    int64_t batch_stride, int box_cols, int box_rows, const char *what);

// ---- layout of a call's workspace -------------------------------------------------------------------------------------------
// Dynamic shared memory that calls of a kernel ask for at most, said once a device.  One number a kernel: threads that say it at once say the same, and
// none takes back what another's launch needs.
template <auto KERNEL, int BYTES>
int allow_smem(const char *what) {
  static std::atomic<bool> allowed[64];
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && (device < 0 || device >= 64 || !allowed[device].load(std::memory_order_relaxed))) {
    e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
    if (e == cudaSuccess && device >= 0 && device < 64) allowed[device].store(true, std::memory_order_relaxed);
  }
  return e == cudaSuccess ? CMACE_OK : fail(CMACE_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct Carve {   // consecutive pieces of the workspace; without a base it only counts
  char *base;
  int64_t used = 0;
  template <typename T>
  T *take(int64_t n) {
    char *p = base ? base + used : nullptr;
    used += up(n * (int64_t)sizeof(T), 256);
    return reinterpret_cast<T *>(p);
  }
};

// Matrices [batches][rows][cols] as operands of the products, rows ld elements apart; pairs as [batches][hi, lo][rows][cols].
struct Matrix {
  CUtensorMap map;         // read in boxes of 64 x 64
  uint16_t *at = nullptr;
  float *scale = nullptr;  // inverse scales of the pairs' blocks, [batches][blocks_m][blocks_n]
  int64_t rows = 0, ld = 0, batches = 1;
  int cols = 0, terms = 1, z0 = 0;
  int64_t blocks_m() const { return (rows + 63) / 64; }
  int64_t blocks_n() const { return (cols + 63) / 64; }
  int64_t plane() const { return rows * ld; }   // elements of a matrix
  Matrix part(int p) const {                    // one of the batches
    Matrix m = *this;
    m.batches = 1, m.z0 = z0 + p * terms;
    if (scale) m.scale = scale + p * blocks_m() * blocks_n();
    return m;
  }
};
inline int encode_matrix(CUtensorMap *map, const Matrix &m, int box_cols, int box_rows, bool bf16, const char *what) {
  return encode_tile_map(map, m.at, 2, bf16, m.cols, m.rows, m.batches * m.terms, m.ld, m.plane(), box_cols, box_rows, what);
}
// in the workspace, rows of a multiple of `align` elements; pairs with or without scales of their blocks
inline Matrix new_matrix(Carve &w, bool pair, int64_t rows, int cols, int64_t batches, int align = 8, bool scales = true) {
  Matrix m;
  m.rows = rows, m.cols = cols, m.batches = batches, m.ld = up(cols, align), m.terms = pair ? 2 : 1;
  m.at = w.take<uint16_t>(batches * m.terms * m.plane());
  if (pair && scales) m.scale = w.take<float>(batches * m.blocks_m() * m.blocks_n());
  return m;
}
// k_inner: the contracted index runs along a row
inline void set_operand(TpOperand &o, const Matrix &m, bool k_inner) {
  o.map = m.map;
  o.mn_major = !k_inner;
  o.z0 = m.z0, o.zstep = m.batches > 1 ? m.terms : 0;
  o.scale = m.scale;
  o.sc_i = k_inner ? m.blocks_n() : 1;
  o.sc_k = k_inner ? 1 : m.blocks_n();
  o.sc_b = m.batches > 1 ? m.blocks_m() * m.blocks_n() : 0;
}

inline TpArgs new_args(int64_t rows, int64_t cols, int32_t *status) {
  TpArgs g;
  memset(&g, 0, sizeof(g));
  g.rows = rows, g.cols = cols, g.status = status;
  g.segments = g.batches = g.splits = 1;
  return g;
}
inline int blocks64(int64_t n) { return (int)((n + 63) / 64); }
inline void set_k(TpArgs &g, int seg, int64_t k) {
  g.kblocks[seg] = blocks64(k);
  g.last16[seg] = (int)((k - 1) % 64) / 16 + 1;
}

// What a variant costs in cycles: rounds of its tiles over the SMs, each as long as its products or, at 50 bytes a cycle and SM, its copies,
// and something for the epilogue and the chain at a tile's ends.  n: columns of B, out: of the output, tn: of a tile.
struct TpCost {
  int64_t rows, out;
  int kblocks;
  int64_t times;
  bool pair;
  int64_t operator()(int ctas, int tn, int n) const {
    const int64_t tiles = (rows + 128 * ctas - 1) / (128 * ctas) * ((out + tn - 1) / tn) * times;
    const int64_t rounds = (tiles + 148 / ctas - 1) / (148 / ctas);
    const int64_t products = (pair ? 3 : 1) * 2 * n, copies = (pair ? 2 : 1) * (128 + n / ctas) * 128 / 50;   // a block of 64 k
    return rounds * (kblocks * (products > copies ? products : copies) + 2000 + 16 * n);
  }
};

// kernels that the dense operators have launched, from any thread
inline std::atomic<int64_t> &dense_launches() {
  static std::atomic<int64_t> count{0};
  return count;
}
template <typename... Params, typename... Args>
void launch_dense(void (*kernel)(Params...), dim3 grid, int threads, cudaStream_t st, Args &&...args) {
  launch_chained(kernel, grid, dim3((unsigned)threads), (size_t)0, st, std::forward<Args>(args)...);
  dense_launches().fetch_add(1, std::memory_order_relaxed);
}
// launch_chained() with clusters of `ctas`
template <typename Args>
int launch_cluster(void (*kernel)(Args), int ctas, int64_t blocks, int threads, int smem, cudaStream_t st, const char *what, const Args &args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  const bool chained = chain_launches() == Chain::on;
  if (chain_launches() == Chain::from_second) chain_launches() = Chain::on;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = ctas > 1 ? attr : attr + 1;
  cfg.numAttrs = (ctas > 1 ? 1 : 0) + (chained ? 1 : 0);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args);
  dense_launches().fetch_add(1, std::memory_order_relaxed);
  return e == cudaSuccess ? check_launch(what) : fail(CMACE_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

template <int KIND, bool PAIR, int TN, int CTAS, int ACT = TP_SILU>
int tp_launch(TpArgs &g, cudaStream_t st, const char *what) {
  using S = TpShape<KIND, PAIR, TN, CTAS>;
  static_assert(S::STAGES >= 2, "a ring of two stages at least");
  g.mt = (int)((g.rows + 128 * CTAS - 1) / (128 * CTAS));
  g.nt = (int)((g.cols + TN - 1) / TN);
  g.total = (int64_t)g.mt * g.nt * g.batches * g.splits;
  if (g.total >= (int64_t)1 << 31) return fail(CMACE_ERR_UNSUPPORTED, "%s: too many tiles", what);
  g.by_nt = tp_div((uint32_t)g.nt), g.by_mt = tp_div((uint32_t)g.mt), g.by_batches = tp_div((uint32_t)g.batches), g.by_splits = tp_div((uint32_t)g.splits);
  const auto kernel = tile_product_kernel<KIND, PAIR, TN, CTAS, ACT>;
  if (const int rc = allow_smem<tile_product_kernel<KIND, PAIR, TN, CTAS, ACT>, S::SMEM>(what)) return rc;
  return launch_cluster(kernel, CTAS, (int)(CTAS * (g.total < 148 / CTAS ? g.total : 148 / CTAS)), TP_THREADS, S::SMEM, st, what, g);
}

}  // namespace cmace
