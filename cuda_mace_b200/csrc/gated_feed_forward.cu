// The gated feed-forward block y = (act(x Wg) * (x Wu)) Wd on rows of node features, and its backward.  x [M, C], Wg and Wu [C, H],
// Wd [H, C], act = SiLU or GELU (with erf).
//
//   forward   h = act(x Wg) * (x Wu)          one kernel: both projections are one product with 256 columns a tile, the gate is
//             y = h Wd                        applied to the accumulators; h [M, H] goes out once, in the operands' form
//   backward  g, u as above, dh = dy Wd^T     one kernel: three products a tile, h, dg = dh u act'(g) and du = dh act(g) out
//             dx = dg Wg^T + du Wu^T          one product over 2 H
//             dWg = x^T dg, dWu = x^T du, dWd = h^T dy    one launch of three products over M, split where M is long
// What bounds them (B200, us alone, cold): widths 1 024 and 4 096, 8 192 rows of bf16: the gated kernel 88 (1 560 TFLOP/s), h Wd 52, the
// backward's hidden values 178 (1 160: 56 bytes of operands for 48 of products a cycle, and 200 MB put down), dx 96, dW 97 + 51; float32 as
// pairs: 283, 152, 540, 298, 306 + 149 (1 350 to 1 450 TFLOP/s of fp16 products), operands 37 before the first and 71 before the third.  Widths
// 128 and 512, 64 000 rows: K is two blocks long, so the elementwise epilogue bounds the first and third: 30, 17, 68, 27, 37 in bf16, 63, 32, 149, 54,
// 74 in float32, where h goes out at 2.1 and h, dg, du at 2.6 TB/s; operands take 14 before the first and 43 before the third.
// Only x and the weights are kept for the backward: forming g and u again costs 4 M C H operations, keeping them in float32 16 bytes
// a hidden value written and read (what would be as exact as the products are), which pays from C of about 1 000 only.
//
// Where tiles would be empty or the chain of kernels long, the forward pass goes another way: few_rows_kernel (up to eight rows) and some_rows_kernel
// (up to 128 columns) below.
// float32 goes as pairs of fp16 values (tile_product.cuh); a first kernel splits x and the weights.  bf16 is read where it lies;
// rows that TMA cannot address (a width that is not a multiple of eight, an address that is not one of 16 bytes) are copied first.
// In bf16, h, dg and du are rounded once to bf16 between the products, as the operands of a 16-bit product have to be; with the
// rounding of the results that makes 1.4 times the error of a result that is rounded alone.  Sums over M are float32.
#include <algorithm>
#include <type_traits>

#include "tile_product.cuh"

namespace cmace {

// ---- operands: float32 to pairs, bf16 rows to rows of a multiple of 16 bytes ------------------------------------------------
struct PrepJob {
  const void *src;
  void *hi, *lo;       // lo null: copy
  float *scale;        // inverse scales of the blocks
  int64_t rows, first; // first block of this job
  int cols, ld, blocks_n, bf16;   // bf16: of the source of a pair
};
// Rows of x, and going back of dL/dy, as pairs.  A block of 64 x 64 values has one scale, under which a row far below the largest is zeros, and
// h goes with the square of a small row.  So the rows of 64 are brought to one size before they are split, each by a power of two: x~ = x / s, dy~ = dy / t.
// A product's rows follow, and what is linear in them: h~ = h / s^2 = g~ sigmoid(g~ s) u~ (SiLU), dg~ = dg / (s t), du~ = du / (s t); y = (h~ Wd) s^2 and
// dx = (..) s t at the end.  A sum over rows has each at the size of its contribution: dWg = (x s t)^T dg~, dWu = (x s t)^T du~,
// dWd = h~^T (dy s^2), for which x and dy are laid out a second time.
// The one size is the mean of the rows' exponents: a row of 1e30, whose own h is no float32 value, then leaves the other rows' h~ where it was.
struct RowsJob {
  const void *src[2];   // x, dy or null
  __half *hi[4];        // x~, dy~, x s t, dy s^2 (null: not wanted), the lo parts a plane behind
  float *scale[4], *size[2];   // inverse scales of the blocks; s and t, ones behind the last row up to a multiple of 256
  float *most[2];       // largest finite magnitudes of the rows' slabs, [slabs][rows]; null: rows of up to two blocks of columns, which a CTA has whole
  int64_t rows, plane, blocks;   // blocks: CTAs
  int cols, ld, blocks_n, bf16, wide, sources, slabs, slab;   // slab: columns
};
struct PrepArgs {
  PrepJob job[5];
  RowsJob rows;
  int jobs;
};
constexpr int PREP_THREADS = 256;

// Four values of a row, zeros for those that are not among the n that it still has.  wide: rows start on 16 bytes.
__device__ __forceinline__ float4 prep_load(const void *src, int64_t at, int n, bool bf16, bool wide) {
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (wide) {
    if (n > 0) x = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(src) + at));
  } else if (bf16) {
    const __nv_bfloat16 *s = static_cast<const __nv_bfloat16 *>(src) + at;
    if (n > 0) x.x = __bfloat162float(s[0]);
    if (n > 1) x.y = __bfloat162float(s[1]);
    if (n > 2) x.z = __bfloat162float(s[2]);
    if (n > 3) x.w = __bfloat162float(s[3]);
  } else {
    const float *s = static_cast<const float *>(src) + at;
    if (n > 0) x.x = __ldg(s);
    if (n > 1) x.y = __ldg(s + 1);
    if (n > 2) x.z = __ldg(s + 2);
    if (n > 3) x.w = __ldg(s + 3);
  }
  return x;
}
__device__ __forceinline__ float prep_most(float4 x) {
  return fmaxf(fmaxf(tp_finite_abs(x.x), tp_finite_abs(x.y)), fmaxf(tp_finite_abs(x.z), tp_finite_abs(x.w)));
}
__device__ __forceinline__ float4 times(float4 x, float f) { return make_float4(x.x * f, x.y * f, x.z * f, x.w * f); }

constexpr int PREP_SLABS = 16;
// A thread has four columns of every 16th row of a block of 64 x 64.
struct PrepThread {
  int64_t row0;
  int first, in, n;   // its first row and column, rows of the block
  __device__ __forceinline__ PrepThread(int t, int64_t row0, int64_t rows)
      : row0(row0), first(t >> 4), in(4 * (t & 15)), n((int)(rows - row0 < 64 ? rows - row0 : 64)) {}
  __device__ __forceinline__ void fetch(float4 (&x)[4], const void *src, int col, int cols, bool bf16, bool wide) const {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = prep_load(src, (row0 + first + 16 * i) * cols + col, first + 16 * i < n ? cols - col : 0, bf16, wide);
  }
};
__device__ __forceinline__ void prep_row_most(float (&most)[4]) {   // of the 16 lanes that have a row
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], d));
}

// Largest finite magnitudes of 64 rows' slabs of columns
__global__ void __launch_bounds__(PREP_THREADS) row_most_kernel(const RowsJob R) {
  grid_begin();
  const PrepThread T(threadIdx.x, (int64_t)blockIdx.x * 64, R.rows);
  const int k = blockIdx.z, end = min(R.cols, (int)(blockIdx.y + 1) * R.slab);
  float most[4] = {};
#pragma unroll 4
  for (int col = (int)blockIdx.y * R.slab + T.in; col < end; col += 64) {
    float4 x[4];
    T.fetch(x, R.src[k], col, R.cols, R.bf16, R.wide);
#pragma unroll
    for (int i = 0; i < 4; i++) most[i] = fmaxf(most[i], prep_most(x[i]));
  }
  prep_row_most(most);
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (T.in == 0 && T.first + 16 * i < T.n) R.most[k][blockIdx.y * R.rows + T.row0 + T.first + 16 * i] = most[i];
}

// COPY: 64 x 64 bf16 values.  Otherwise pairs: a block of a weight, or one block of x or dy (BLOCKS), or 64 rows of x (WHOLE) or of x and dy (BOTH, a
// half of the threads each) of up to 128 columns, whose sizes the CTA finds itself: 64 000 rows of 128, x and dy: 43 us, by blocks
// and a kernel for the sizes 54.
enum PrepKind { PREP_COPY, PREP_WHOLE, PREP_BOTH, PREP_BLOCKS };
constexpr int prep_threads(int kind) { return (kind == PREP_BOTH ? 2 : 1) * PREP_THREADS; }
template <int KIND>
__global__ void __launch_bounds__(prep_threads(KIND), KIND == PREP_COPY ? 8 : KIND == PREP_WHOLE ? 4 : KIND == PREP_BOTH ? 2 : 5)
    prep_kernel(const __grid_constant__ PrepArgs p) {
  constexpr bool ROWS = KIND == PREP_WHOLE || KIND == PREP_BOTH;
  constexpr int NB = ROWS ? 2 : 1;                         // blocks of a CTA
  __shared__ float most_of[2][NB][2][PREP_THREADS / 32];   // of both sources and layouts
  __shared__ int sum_of[2][PREP_THREADS / 32], top_of[2][PREP_THREADS / 32], exponent_of[2][64];
  grid_begin();
  const RowsJob &R = p.rows;
  const bool rows = KIND != PREP_COPY && (int64_t)blockIdx.x < R.blocks;
  int j = 0;
  while (j + 1 < p.jobs && (int64_t)blockIdx.x >= p.job[j + 1].first) j++;
  const PrepJob &J = p.job[j];
  const int across = rows ? (ROWS ? 1 : R.blocks_n * R.sources) : J.blocks_n, t = threadIdx.x % PREP_THREADS, half = threadIdx.x / PREP_THREADS;
  const int64_t b = rows ? blockIdx.x : blockIdx.x - J.first, rb = b / across;
  int cb = (int)(b - rb * across);
  if constexpr (KIND == PREP_COPY) {
    const uint16_t *s = static_cast<const uint16_t *>(J.src);
    uint16_t *d = static_cast<uint16_t *>(J.hi);
    const int64_t row0 = rb * 64;
    const int col = 64 * cb + (t & 63);
    if (col < J.cols)
      for (int r = t >> 6; r < 64 && row0 + r < J.rows; r += 4) d[(row0 + r) * J.ld + col] = s[(row0 + r) * J.cols + col];
    return;
  }
  if (!rows && half) return;
  const int k = KIND == PREP_BOTH ? half : KIND == PREP_BLOCKS && rows && R.sources == 2 ? cb & 1 : 0;   // x or dy
  if (KIND == PREP_BLOCKS && rows && R.sources == 2) cb >>= 1;
  const PrepThread T(t, rb * 64, rows ? R.rows : J.rows);
  const int warp = t >> 5, cols = rows ? R.cols : J.cols, ld = rows ? R.ld : J.ld, blocks = ROWS && rows ? R.blocks_n : 1;
  const bool bf16 = rows ? R.bf16 : J.bf16, wide = rows ? R.wide : (cols & 3) == 0 && (reinterpret_cast<uintptr_t>(J.src) & 15) == 0 && !bf16;
  float4 x[NB][4];
#pragma unroll
  for (int e = 0; e < NB; e++)
    if (e < blocks) T.fetch(x[e], rows ? R.src[k] : J.src, 64 * (cb + e) + T.in, cols, bf16, wide);
  // The sizes of this thread's rows, its own ([0]) and the other source's, by the exponents of the rows' largest finite values
  constexpr int NONE = 1 << 20;
  int below[2][4] = {};   // exponents with float32's bias, then how far below the group's mean (126 at most); NONE: a row of zeros
  const auto exp2i = [](int e) { return __uint_as_float((uint32_t)(e + 127) << 23); };   // -126 <= e <= 127
  if (rows) {
#pragma unroll
    for (int o = 0; o < (ROWS ? 1 : 2); o++) {
      if (o >= R.sources) break;
      float most[4] = {};
      if constexpr (ROWS) {
#pragma unroll
        for (int e = 0; e < NB; e++) {
          if (e >= blocks) break;
#pragma unroll
          for (int i = 0; i < 4; i++) most[i] = fmaxf(most[i], prep_most(x[e][i]));
        }
      } else if ((t & 15) < R.slabs) {
        const float *from = R.most[o ? 1 - k : k] + (t & 15) * R.rows + T.row0 + T.first;
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (T.first + 16 * i < T.n) most[i] = __ldcg(from + 16 * i);
      }
      prep_row_most(most);
      int sum = 0;   // and the number of them, above
#pragma unroll
      for (int i = 0; i < 4; i++) {
        below[o][i] = most[i] == 0.f ? NONE : (int)(__float_as_uint(most[i]) >> 23);
        if (T.in == 0 && below[o][i] != NONE) sum += below[o][i] + (1 << 16);
        if (KIND == PREP_BOTH && T.in == 0) exponent_of[k][T.first + 16 * i] = below[o][i];
      }
      sum = __reduce_add_sync(0xffffffffu, sum);
      if ((t & 31) == 0) sum_of[o ? 1 - k : k][warp] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int o = 0; o < (KIND == PREP_WHOLE ? 1 : 2); o++) {
      if (o >= R.sources) break;
      int sum = 0;
#pragma unroll
      for (int w = 0; w < PREP_THREADS / 32; w++) sum += sum_of[o ? 1 - k : k][w];
      const int count = max(sum >> 16, 1), mean = ((sum & 0xFFFF) + count / 2) / count;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (KIND == PREP_BOTH && o) below[o][i] = exponent_of[1 - k][T.first + 16 * i];
        if (below[o][i] != NONE) below[o][i] = min(max(mean - below[o][i], -126), 126);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (cb == 0 && T.in == 0 && T.first + 16 * i < T.n) R.size[k][T.row0 + T.first + 16 * i] = below[0][i] == NONE ? 1.f : exp2i(-below[0][i]);
    if (cb == 0 && T.row0 + 64 >= R.rows && R.rows + t < (R.rows + 255) / 256 * 256) R.size[k][R.rows + t] = 1.f;
  }
  // As a contribution, x s t or dy s^2, below the group's largest s t or s^2.  A row of zeros contributes nothing, whatever the other has.
  int less[4] = {}, top = -NONE;
  if (KIND != PREP_WHOLE && rows && R.sources == 2) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int own = below[0][i], other = below[1][i];
      less[i] = own == NONE || other == NONE ? -NONE : k ? -2 * other : -own - other;
      top = max(top, less[i]);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((t & 31) == 0) top_of[half][warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PREP_THREADS / 32; w++) top = max(top, top_of[half][w]);
    if (top == -NONE) top = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) less[i] -= top;
  }
  const auto twice = [&](int e) { return make_float2(exp2i(e / 2), exp2i(e - e / 2)); };   // 2^e as two factors, |e| <= 252
  const auto value = [&](const float4 &v, int how, int i) {
    if (how == 0) return times(v, below[0][i] == NONE ? 1.f : exp2i(below[0][i]));
    const float2 f = less[i] < -252 ? make_float2(0.f, 0.f) : twice(less[i]);
    return times(times(v, f.x), f.y);
  };
  __half *const hi[2] = {rows ? R.hi[k] : static_cast<__half *>(J.hi), KIND != PREP_WHOLE && rows ? R.hi[2 + k] : nullptr};
#pragma unroll
  for (int e = 0; e < NB; e++)
#pragma unroll
    for (int how = 0; how < 2; how++) {
      if (e >= blocks || !hi[how]) continue;
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < 4; i++) most = fmaxf(most, prep_most(value(x[e][i], how, i)));
      most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
      if ((t & 31) == 0) most_of[half][e][how][warp] = most;
    }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < NB; e++)
#pragma unroll
    for (int how = 0; how < 2; how++) {
      if (e >= blocks || !hi[how]) continue;
      float most = most_of[half][e][how][0];
#pragma unroll
      for (int w = 1; w < PREP_THREADS / 32; w++) most = fmaxf(most, most_of[half][e][how][w]);
      const float scale = tp_scale(most);
      if (t == 0) {
        const float2 f = how ? twice(top) : make_float2(1.f, 1.f);
        (rows ? R.scale[2 * how + k] + rb * R.blocks_n + cb + e : J.scale + b)[0] = 1.0f / scale * f.x * f.y;
      }
      const int col = 64 * (cb + e) + T.in;
      __half *const to = hi[how] + (T.row0 + T.first) * ld + col, *const to_lo = to + (rows ? R.plane : static_cast<__half *>(J.lo) - hi[how]);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (T.first + 16 * i >= T.n || col >= cols) break;   // columns up to the rows' distance, a multiple of eight, take zeros
        const float4 v = value(x[e][i], how, i);
        uint2 h, l;
        tp_split2(v.x, v.y, scale, h.x, l.x);
        tp_split2(v.z, v.w, scale, h.y, l.y);
        *reinterpret_cast<uint2 *>(to + (int64_t)(16 * i) * ld) = h;
        *reinterpret_cast<uint2 *>(to_lo + (int64_t)(16 * i) * ld) = l;
      }
    }
}

// ---- few rows: a pass over the weights -------------------------------------------------------------------------------------------
// With up to eight rows the block is as long as its weights take to arrive, and a tensor core's tile would be 1/16 full at most: plain
// float32 FMA, a weight read once for all rows.  A CTA has 32 columns (segments of 64 or 128 bytes of a row), its 16 warps every 64th group
// of rows of W, and the CTAs of a cluster share the rows where columns alone do not fill the SMs.  h stays float32 in the workspace.
// Three sets of weights in turn, both kernels in a recorded graph, us: 1 024 and 4 096, one row 9.5 in bf16 and 14.5 in float32, eight rows 21 and 24
// against 20.5 and 44 by tiles; 512 and 2 048, one row 10 and 9.6 (clusters), eight 15.5 and 15 against 15.5 and 27.  Eight rows are bound by
// FMA and by their operands: x from shared memory, weights to float32.
constexpr int FEW_ROWS = 8, FEW_THREADS = 512, FEW_COLS = 32, FEW_K = 1024;   // FEW_K: rows of W whose x is in shared memory

struct FewArgs {
  const void *x;       // [M, K]: T, or h in float32
  const void *w[2];    // [K, N]
  void *out;           // [M, N]: h in float32, or T
  int M, K, N, cluster, wide;
  int32_t *status;
};

// V values from p as they lie, the first n of them (wide: all, aligned), zeros for the others
template <typename T, int V, int WORDS = V * (int)sizeof(T) / 4>
__device__ __forceinline__ void few_load(uint32_t (&v)[WORDS], const T *p, int n, bool wide) {
  if (wide) {
    if constexpr (WORDS == 4) {
      const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p));
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
      const uint2 x = __ldg(reinterpret_cast<const uint2 *>(p));
      v[0] = x.x, v[1] = x.y;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = i < n ? __float_as_uint(__ldg(p + i)) : 0u;
  } else {
    const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
    for (int i = 0; i < WORDS; i++) v[i] = (2 * i < n ? (uint32_t)__ldg(h + 2 * i) : 0u) | (2 * i + 1 < n ? (uint32_t)__ldg(h + 2 * i + 1) << 16 : 0u);
  }
}
template <typename T, int WORDS>
__device__ __forceinline__ float few_value(const uint32_t (&v)[WORDS], int i) {
  if (sizeof(T) == 4) return __uint_as_float(v[i % WORDS]);
  const uint32_t w = v[i / 2];
  return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
}
// columns a thread: 16 bytes, 8 where the sums of eight rows would not fit the registers
template <typename T, int M>
constexpr int few_cols() { return sizeof(T) == 2 && M <= 4 ? 8 : 4; }

// GATED: h = act(x Wg) * (x Wu), otherwise y = h Wd.  M: rows, or up to seven more.
template <typename T, int M, bool GATED, int ACT>
__global__ void __launch_bounds__(FEW_THREADS, 1) few_rows_kernel(const FewArgs g) {
  constexpr int W = GATED ? 2 : 1, WARPS = FEW_THREADS / 32, V = few_cols<T, M>(), LANES = FEW_COLS / V, ROWS = 32 / LANES;   // of a warp's load
  extern __shared__ float few_smem[];   // x [FEW_K][M]; then the warps' sums [WARPS][W][M][32]
  __shared__ float total[8][W][M][FEW_COLS];   // of the CTAs of a cluster, in the first one's
  __shared__ __align__(8) uint64_t joined;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane % LANES, row = lane / LANES;
  const int rank = blockIdx.x % g.cluster, col = (int)(blockIdx.x / g.cluster) * FEW_COLS + V * part;
  const int k0 = (int)((int64_t)g.K * rank / g.cluster), k1 = (int)((int64_t)g.K * (rank + 1) / g.cluster);
  const int n = g.N - col;
  if (g.cluster > 1) {
    if (threadIdx.x == 0) {
      mbar_init(smem_u32(&joined), (uint32_t)g.cluster - 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    cluster_arrive();
  }
  // Wd does not come from the kernel before: it is on its way while that one ends.
  if (!GATED) {
    const T *w = static_cast<const T *>(g.w[0]) + (int)(blockIdx.x / g.cluster) * FEW_COLS;
    for (int k = k0 + (int)threadIdx.x; k < k1; k += FEW_THREADS) asm volatile("prefetch.global.L1 [%0];" ::"l"(w + (int64_t)k * g.N));
  }
  grid_begin();
  float acc[W][M][V] = {};
  for (int from = k0; from < k1; from += FEW_K) {
    const int len = min(FEW_K, k1 - from);
    __syncthreads();
    for (int i = threadIdx.x; i < len * M; i += FEW_THREADS) {
      const int m = i / len, k = i - m * len;
      float v = 0.f;
      if (m < g.M) {
        const int64_t at = (int64_t)m * g.K + from + k;
        v = GATED ? (float)static_cast<const T *>(g.x)[at] : __ldcg(static_cast<const float *>(g.x) + at);   // h: of the kernel before
      }
      few_smem[k * M + m] = v;
    }
    __syncthreads();
    if (n > 0) {
      // AHEAD loads leave together, however long the rest is; behind the last row they read it once more,
      // for nothing.
      constexpr int AHEAD = M <= 2 ? 8 : 4, STEP = ROWS * WARPS;
      for (int first = ROWS * warp + row; first < len; first += AHEAD * STEP) {
        uint32_t w[AHEAD][W][V * (int)sizeof(T) / 4];
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
          if (first - row + a * STEP >= len) break;   // none of the warp's rows
#pragma unroll
          for (int i = 0; i < W; i++)
            few_load<T, V>(w[a][i], static_cast<const T *>(g.w[i]) + (int64_t)(from + min(first + a * STEP, len - 1)) * g.N + col, n, g.wide);
        }
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
          if (first + a * STEP >= len) break;
          float x[M];
#pragma unroll
          for (int m = 0; m < M; m++) x[m] = few_smem[(first + a * STEP) * M + m];
#pragma unroll
          for (int i = 0; i < W; i++)
#pragma unroll
            for (int m = 0; m < M; m++)
#pragma unroll
              for (int j = 0; j < V; j++) acc[i][m][j] = fmaf(x[m], few_value<T>(w[a][i], j), acc[i][m][j]);
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; i++)
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
      for (int j = 0; j < V; j++) {
        float v = acc[i][m][j];
#pragma unroll
        for (int d = LANES; d < 32; d *= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
        if (row == 0) few_smem[((warp * W + i) * M + m) * FEW_COLS + V * part + j] = v;
      }
  __syncthreads();
  // The first CTA of a cluster gets the others' sums: one arrival each instead of two barriers of all threads: 11.1 us for a row of
  // 512 x 2 048 in bf16, 12.0 with those.
  if (g.cluster > 1) {
    __syncwarp();
    cluster_wait();
  }
  for (int e = threadIdx.x; e < W * M * FEW_COLS; e += FEW_THREADS) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; k++) v += few_smem[k * (W * M * FEW_COLS) + e];
    float *const to = &total[rank][0][0][0] + e;
    if (rank == 0) *to = v;
    else asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(peer_smem(smem_u32(to), 0)), "f"(v) : "memory");
  }
  __syncthreads();
  if (rank != 0) {
    if (threadIdx.x == 0) peer_arrive(smem_u32(&joined), 0);
    return;
  }
  if (g.cluster > 1 && !peer_wait(smem_u32(&joined), 0) && g.status) atomicCAS(g.status, 0, 112);
  for (int e = threadIdx.x; e < M * FEW_COLS; e += FEW_THREADS) {
    const int m = e / FEW_COLS, c = (int)(blockIdx.x / g.cluster) * FEW_COLS + e % FEW_COLS;
    float v[W];
#pragma unroll
    for (int i = 0; i < W; i++) {
      v[i] = 0.f;
      for (int r = 0; r < g.cluster; r++) v[i] += total[r][i][m][e % FEW_COLS];
    }
    if (m < g.M && c < g.N) {
      if (GATED) static_cast<float *>(g.out)[(int64_t)m * g.N + c] = tp_act<ACT>(v[0]) * v[W - 1];
      else static_cast<T *>(g.out)[(int64_t)m * g.N + c] = (T)v[0];
    }
  }
}

// ---- some rows: the whole block in one kernel -----------------------------------------------------------------------------------
// Where few tiles are full, a call is as long as its chain of kernels (copies, products, an epilogue, the next kernel's start: 5 to 6 us each),
// and a full tile's tensor-core rate counts for nothing.
// Here a warp needs nobody until the end: it has 16 rows and a group of 16 (float32) or 32 (bf16) hidden columns, forms g and u of them
// with warp-wide MMAs (mma.sync), and multiplies h, whose sums lie in the registers as the next product's operand has to, with its rows of Wd.
// Weights come from L2 to registers once a block of 16 rows, four k a lane: k and the columns are dealt to lanes so that a lane's
// loads are vectors (the order of k in a product is free).  The warps' sums of y are added at the end, in shared memory and over a
// cluster that shares the hidden columns, in one order.  float32: three products of TF32 parts (lo hi, hi lo, hi hi) of 16 k, started at zero and
// added to float32 registers, so that the tensor core's truncation stays at 2^-24 of a partial sum.
// 192 rows, 128 and 512: float32 12 us against 17.7 by tiles, bf16 9.0 against 10.7; 400 rows, 32 and 512: 5.9 against 16.1, 5.3 against 10.2.  A
// warp's chain bounds it (loads, six dependent products a step, 16 values a load to split): two rows of blocks an SM at once do not fit the
// registers.  Groups spread over twice as many CTAs: the same (a cluster costs 1.7; sums pushed to the CTA that stores them, with one arrival each: the same or 1 more).
constexpr int SOME_THREADS = 256, SOME_WARPS = SOME_THREADS / 32, SOME_ROWS = 16;

struct SomeArgs {
  const void *x, *w[2], *wd;
  void *y;
  int64_t M;
  int C, H, ld, cluster, wide;   // ld: elements a row of x in shared memory
};
constexpr int some_group(bool f32) { return f32 ? 16 : 32; }   // hidden columns

__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// x = hi + lo to 2^-22 of x, both rounded to TF32's 11 bits
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}
// two values as bf16 and what that leaves: h keeps 16 bits, for half as many products again
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t &hi, uint32_t &lo) {
  hi = tp_bf16x2(x, y);
  lo = tp_bf16x2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xFFFF0000u));
}
// 8 or 16 bytes of `base`, `off` bytes behind it (the matrices here are below 4 GB).  FULL: all of it is there and aligned.  Otherwise the
// first n elements are (WIDE: all or none, aligned), zeros stand for the others, and their loads go to the matrix's first elements: loads
// without a branch leave together.
template <typename T, bool FULL, bool WIDE, int WORDS>
__device__ __forceinline__ void some_load(uint32_t (&v)[WORDS], const void *base, uint32_t off, int n) {
  const char *p = static_cast<const char *>(base);
  if constexpr (FULL || WIDE) {
    p += FULL || n > 0 ? off : 0u;
    if constexpr (WORDS == 4) {
      const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p));
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
      const uint2 x = __ldg(reinterpret_cast<const uint2 *>(p));
      v[0] = x.x, v[1] = x.y;
    }
    if (FULL) return;
#pragma unroll
    for (int i = 0; i < WORDS; i++) v[i] = n > 0 ? v[i] : 0u;
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < WORDS; i++) {
      const uint32_t x = __ldg(reinterpret_cast<const uint32_t *>(p + (i < n ? off + 4 * i : 0u)));
      v[i] = i < n ? x : 0u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; i++) {
      const uint32_t x = __ldg(reinterpret_cast<const uint16_t *>(p + (2 * i < n ? off + 4 * i : 0u)));
      const uint32_t y = __ldg(reinterpret_cast<const uint16_t *>(p + (2 * i + 1 < n ? off + 4 * i + 2 : 0u)));
      v[i] = (2 * i < n ? x : 0u) | (2 * i + 1 < n ? y << 16 : 0u);
    }
  }
}
// the two k of column t of a bf16 operand, from two rows' words
__device__ __forceinline__ uint32_t k_pair(const uint32_t (&a)[2], const uint32_t (&b)[2], int t) {
  return __byte_perm(a[t >> 1], b[t >> 1], t & 1 ? 0x7632 : 0x5410);
}

// a lane's columns col, col + 1, ... of both projections, of rows k .. k + 3 and those of the next steps of 16
template <typename T, bool FULL, bool WIDE, int DEPTH>
__device__ __forceinline__ void some_projections(uint32_t (&to)[DEPTH][2][4][2], const SomeArgs &g, int col, int k) {
  const uint32_t row = (uint32_t)(g.H * (int)sizeof(T));
  uint32_t off = (uint32_t)k * row + (uint32_t)(col * (int)sizeof(T));
#pragma unroll
  for (int d = 0; d < DEPTH; d++, off += 12 * row)
#pragma unroll
    for (int i = 0; i < 4; i++, off += row)
#pragma unroll
      for (int p = 0; p < 2; p++) some_load<T, FULL, WIDE>(to[d][p][i], g.w[p], off, k + 16 * d + i < g.C ? g.H - col : 0);
}
// columns col .. col + 3 of Wd's rows: the hidden columns k + t and k + NT + t that a lane has values of
template <typename T, bool FULL, bool WIDE, int NT, int DW>
__device__ __forceinline__ void some_down(uint32_t (&to)[NT][2][DW], const SomeArgs &g, int k, int col) {
  const uint32_t row = (uint32_t)(g.C * (int)sizeof(T)), off = (uint32_t)k * row + (uint32_t)(col * (int)sizeof(T));
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int i = 0; i < 2; i++) some_load<T, FULL, WIDE>(to[t][i], g.wd, off + (uint32_t)(NT * i + t) * row, k + NT * i + t < g.H ? g.C - col : 0);
}

// CT: spans of 32 columns of y, at least C / 32
template <typename T, int CT, int ACT>
__global__ void __launch_bounds__(SOME_THREADS, 1) some_rows_kernel(const SomeArgs g) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int GROUP = some_group(F32), NT = GROUP / 8, DEPTH = 2;   // DEPTH: steps of 16 k that are loaded together
  constexpr int COLS = 32 * CT, RED = SOME_ROWS * COLS;
  extern __shared__ __align__(16) unsigned char some_smem[];
  T *const xs = reinterpret_cast<T *>(some_smem);   // x [16][ld], float32: hi, then lo
  float *const red = reinterpret_cast<float *>(some_smem + (F32 ? 2 : 1) * SOME_ROWS * g.ld * (int)sizeof(T));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q = lane & 3, j = lane >> 2;
  const int rank = g.cluster > 1 ? (int)cluster_rank() : 0;
  const int64_t row0 = (int64_t)(blockIdx.x / (unsigned)g.cluster) * SOME_ROWS;
  const int steps = (g.C + 15) / 16, groups = (g.H + GROUP - 1) / GROUP;
  const auto fetch = [&](uint32_t (&to)[DEPTH][2][4][2], int group, int step) {
    const int col = group * GROUP + NT * j, k = 16 * step + 4 * q;
    if (g.wide && (group + 1) * GROUP <= g.H && 16 * (step + DEPTH) <= g.C) some_projections<T, true, true>(to, g, col, k);
    else if (g.wide) some_projections<T, false, true>(to, g, col, k);
    else some_projections<T, false, false>(to, g, col, k);
  };
  constexpr int DW = F32 ? 4 : 2;   // words of four columns of y
  const auto fetch_down = [&](uint32_t (&to)[NT][2][DW], int group, int span) {
    const int k = group * GROUP + 2 * NT * q, col = 32 * span + 4 * j;
    if (g.wide && (group + 1) * GROUP <= g.H && 32 * span + 32 <= g.C) some_down<T, true, true>(to, g, k, col);
    else if (g.wide) some_down<T, false, true>(to, g, k, col);
    else some_down<T, false, false>(to, g, k, col);
  };
  const int first = rank * SOME_WARPS + warp;
  uint32_t w[2][DEPTH][2][4][2];
  fetch(w[0], first, 0);
#pragma unroll
  for (int r = warp; r < SOME_ROWS; r += SOME_WARPS)
    for (int k = 4 * lane; k < 16 * steps; k += 128) {
      constexpr int XW = F32 ? 4 : 2;
      uint32_t v[XW];
      const void *row = static_cast<const T *>(g.x) + (row0 + r < g.M ? row0 + r : row0) * g.C;
      const int n = row0 + r < g.M ? g.C - k : 0;
      if (g.wide) some_load<T, false, true>(v, row, (uint32_t)(k * (int)sizeof(T)), n);
      else some_load<T, false, false>(v, row, (uint32_t)(k * (int)sizeof(T)), n);
      if constexpr (F32) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split_tf32(__uint_as_float(v[i]), hi[i], lo[i]);
        *reinterpret_cast<uint4 *>(xs + r * g.ld + k) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(xs + (SOME_ROWS + r) * g.ld + k) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      } else {
        *reinterpret_cast<uint2 *>(xs + r * g.ld + k) = make_uint2(v[0], v[1]);
      }
    }
  __syncthreads();
  float y[CT][4][4] = {};
  for (int group = first; group < groups; group += g.cluster * SOME_WARPS) {
    float sum[2][NT][4] = {};
    const auto multiply = [&](const uint32_t (&from)[DEPTH][2][4][2], int step) {
#pragma unroll
      for (int d = 0; d < DEPTH; d++) {
        if (step + d >= steps) break;
        const T *a = xs + j * g.ld + 16 * (step + d) + 4 * q;
        if constexpr (F32) {
          const float4 h0 = *reinterpret_cast<const float4 *>(a), h1 = *reinterpret_cast<const float4 *>(a + 8 * g.ld);
          const float4 l0 = *reinterpret_cast<const float4 *>(a + 16 * g.ld), l1 = *reinterpret_cast<const float4 *>(a + 24 * g.ld);
          const uint32_t ah[2][4] = {{__float_as_uint(h0.x), __float_as_uint(h1.x), __float_as_uint(h0.y), __float_as_uint(h1.y)},
                                     {__float_as_uint(h0.z), __float_as_uint(h1.z), __float_as_uint(h0.w), __float_as_uint(h1.w)}};
          const uint32_t al[2][4] = {{__float_as_uint(l0.x), __float_as_uint(l1.x), __float_as_uint(l0.y), __float_as_uint(l1.y)},
                                     {__float_as_uint(l0.z), __float_as_uint(l1.z), __float_as_uint(l0.w), __float_as_uint(l1.w)}};
          // six products of 2 NT sums in turn: each waits for the one before of its sum
          uint32_t bh[2 * NT][4], bl[2 * NT][4];
          float part[2 * NT][4] = {};
#pragma unroll
          for (int n = 0; n < 2 * NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) split_tf32(__uint_as_float(from[d][n / NT][i][n % NT]), bh[n][i], bl[n][i]);
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int n = 0; n < 2 * NT; n++) mma_tf32(part[n], al[e][0], al[e][1], al[e][2], al[e][3], bh[n][2 * e], bh[n][2 * e + 1]);
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int n = 0; n < 2 * NT; n++) mma_tf32(part[n], ah[e][0], ah[e][1], ah[e][2], ah[e][3], bl[n][2 * e], bl[n][2 * e + 1]);
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int n = 0; n < 2 * NT; n++) mma_tf32(part[n], ah[e][0], ah[e][1], ah[e][2], ah[e][3], bh[n][2 * e], bh[n][2 * e + 1]);
#pragma unroll
          for (int n = 0; n < 2 * NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) sum[n / NT][n % NT][i] += part[n][i];
        } else {
          const uint2 a0 = *reinterpret_cast<const uint2 *>(a), a1 = *reinterpret_cast<const uint2 *>(a + 8 * g.ld);
#pragma unroll
          for (int p = 0; p < 2; p++)
#pragma unroll
            for (int t = 0; t < NT; t++)
              mma_bf16(sum[p][t], a0.x, a1.x, a0.y, a1.y, k_pair(from[d][p][0], from[d][p][1], t), k_pair(from[d][p][2], from[d][p][3], t));
        }
      }
    };
    uint32_t down[2][NT][2][DW];
    for (int step = 0; step < steps; step += 2 * DEPTH) {
      if (step + DEPTH < steps) fetch(w[1], group, step + DEPTH);
      multiply(w[0], step);
      if (step + 2 * DEPTH < steps) fetch(w[0], group, step + 2 * DEPTH);
      else fetch_down(down[0], group, 0);
      if (step + DEPTH < steps) multiply(w[1], step + DEPTH);
    }
    // h of column NT (2 q + c) + t: rows j (values 0, 1) and j + 8 (2, 3) of tile t
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) sum[0][t][i] = tp_act<ACT>(sum[0][t][i]) * sum[1][t][i];
#pragma unroll
    for (int span = 0; span < CT; span++) {
      if (span + 1 < CT) fetch_down(down[(span + 1) & 1], group, span + 1);   // spans behind C: of zeros
      else if (group + g.cluster * SOME_WARPS < groups) fetch(w[0], group + g.cluster * SOME_WARPS, 0);
      const uint32_t(&b)[NT][2][DW] = down[span & 1];
      if constexpr (F32) {
        float part[4][4] = {};
        uint32_t ah[NT][4], al[NT][4];   // k of the product: q and q + 4 are columns 2 q and 2 q + 1 of the tile
#pragma unroll
        for (int t = 0; t < NT; t++) {
          split_tf32(sum[0][t][0], ah[t][0], al[t][0]);
          split_tf32(sum[0][t][2], ah[t][1], al[t][1]);
          split_tf32(sum[0][t][1], ah[t][2], al[t][2]);
          split_tf32(sum[0][t][3], ah[t][3], al[t][3]);
        }
        uint32_t bh[4][NT][2], bl[4][NT][2];
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 2; i++) split_tf32(__uint_as_float(b[t][i][s]), bh[s][t][i], bl[s][t][i]);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int s = 0; s < 4; s++) mma_tf32(part[s], al[t][0], al[t][1], al[t][2], al[t][3], bh[s][t][0], bh[s][t][1]);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int s = 0; s < 4; s++) mma_tf32(part[s], ah[t][0], ah[t][1], ah[t][2], ah[t][3], bl[s][t][0], bl[s][t][1]);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int s = 0; s < 4; s++) mma_tf32(part[s], ah[t][0], ah[t][1], ah[t][2], ah[t][3], bh[s][t][0], bh[s][t][1]);
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
          for (int i = 0; i < 4; i++) y[span][s][i] += part[s][i];
      } else {
#pragma unroll
        for (int t = 0; t < NT; t += 2) {
          uint32_t a[4], l[4];
          split_bf16(sum[0][t][0], sum[0][t][1], a[0], l[0]);
          split_bf16(sum[0][t][2], sum[0][t][3], a[1], l[1]);
          split_bf16(sum[0][t + 1][0], sum[0][t + 1][1], a[2], l[2]);
          split_bf16(sum[0][t + 1][2], sum[0][t + 1][3], a[3], l[3]);
#pragma unroll
          for (int s = 0; s < 4; s++) {
            const uint32_t b0 = k_pair(b[t][0], b[t][1], s), b1 = k_pair(b[t + 1][0], b[t + 1][1], s);
            mma_bf16(y[span][s], a[0], a[1], a[2], a[3], b0, b1);
            mma_bf16(y[span][s], l[0], l[1], l[2], l[3], b0, b1);
          }
        }
      }
    }
  }
  // columns 8 q .. 8 q + 7 of a span, of rows j and j + 8
#pragma unroll
  for (int span = 0; span < CT; span++)
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
      for (int c = 0; c < 2; c++)
        *reinterpret_cast<float4 *>(red + warp * RED + (j + 8 * r) * COLS + 32 * span + 8 * q + 4 * c) =
            make_float4(y[span][0][2 * r + c], y[span][1][2 * r + c], y[span][2][2 * r + c], y[span][3][2 * r + c]);
  __syncthreads();
  const auto store = [&](int e, const float4 &v) {
    const int64_t row = row0 + e / COLS;
    const int c = e % COLS, n = row < g.M ? g.C - c : 0;
    T *to = static_cast<T *>(g.y) + row * g.C + c;
    if (g.wide) {
      if (n <= 0) return;
      if constexpr (F32) *reinterpret_cast<float4 *>(to) = v;
      else *reinterpret_cast<uint2 *>(to) = make_uint2(tp_bf16x2(v.x, v.y), tp_bf16x2(v.z, v.w));
    } else {
      if (n > 0) to[0] = (T)v.x;
      if (n > 1) to[1] = (T)v.y;
      if (n > 2) to[2] = (T)v.z;
      if (n > 3) to[3] = (T)v.w;
    }
  };
  for (int e = 4 * tid; e < RED; e += 4 * SOME_THREADS) {
    float4 v = *reinterpret_cast<const float4 *>(red + e);
#pragma unroll
    for (int k = 1; k < SOME_WARPS; k++) {
      const float4 o = *reinterpret_cast<const float4 *>(red + k * RED + e);
      v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
    }
    if (g.cluster == 1) store(e, v);
    else *reinterpret_cast<float4 *>(red + e) = v;
  }
  if (g.cluster == 1) return;
  __syncwarp();
  cluster_sync();
  const int per = RED / g.cluster;
  for (int e = rank * per + 4 * tid; e < (rank + 1) * per; e += 4 * SOME_THREADS) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = 0; r < g.cluster; r++) {
      float4 o;
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(o.x), "=f"(o.y), "=f"(o.z), "=f"(o.w)
                   : "r"(peer_smem(smem_u32(red + e), (uint32_t)r))
                   : "memory");
      v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
    }
    store(e, v);
  }
  __syncwarp();
  cluster_sync();   // nobody leaves while its sums are read
}

// ---- weight gradients: the splits' sums, the third transposed ------------------------------------------------------------------
struct WeightReduce {
  const float *partial;   // [splits][3][C][ld]
  void *out[3];
  int64_t ld;
  int splits, C, H;
};
// A block sums 32 x 32 values of one matrix, in the order of the splits.
template <typename T>
__global__ void __launch_bounds__(256) weight_reduce_kernel(const WeightReduce p) {
  __shared__ float tile[32][33];
  grid_begin();
  const int which = blockIdx.z, c0 = blockIdx.y * 32, h0 = blockIdx.x * 32;
  T *out = static_cast<T *>(p.out[which]);
  if (out == nullptr) return;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t matrix = (int64_t)p.C * p.ld;
  const int h = h0 + x;
  const float *v = p.partial + which * matrix + (int64_t)(c0 + y) * p.ld + h;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (h < p.H) {
#pragma unroll 4
    for (int s = 0; s < p.splits; s++, v += 3 * matrix)
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (c0 + y + 8 * i < p.C) sum[i] += __ldcg(v + (int64_t)(8 * i) * p.ld);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int c = c0 + y + 8 * i;
    if (which < 2 && c < p.C && h < p.H) out[(int64_t)c * p.H + h] = (T)sum[i];
    tile[y + 8 * i][x] = sum[i];
  }
  if (which < 2) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int h = h0 + y + 8 * i, c = c0 + x;
    if (c < p.C && h < p.H) out[(int64_t)h * p.C + c] = (T)tile[x][y + 8 * i];
  }
}

// ---- rows of y or dx whose sum over the hidden columns was split: added in the order of the splits ------------------------------------
struct RowsSum {
  const float *partial;   // [splits][M][ld]
  void *out;              // [M][C]
  int64_t M;
  int ld, C, splits, wide;
};
// A thread adds four columns of a row.
template <typename T>
__global__ void __launch_bounds__(256) rows_sum_kernel(const RowsSum p) {
  grid_begin();
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, plane = p.M * p.ld;
  if (at >= plane) return;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < p.splits; s++) {
    const float4 o = __ldcg(reinterpret_cast<const float4 *>(p.partial + s * plane + at));
    v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
  }
  const int64_t row = at / p.ld;
  const int c = (int)(at - row * p.ld), n = p.C - c;
  T *to = static_cast<T *>(p.out) + row * p.C + c;
  if (p.wide) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(to) = v;
    else *reinterpret_cast<uint2 *>(to) = make_uint2(tp_bf16x2(v.x, v.y), tp_bf16x2(v.z, v.w));
  } else {
    to[0] = (T)v.x;
    if (n > 1) to[1] = (T)v.y;
    if (n > 2) to[2] = (T)v.z;
    if (n > 3) to[3] = (T)v.w;
  }
}

// ---- a call -----------------------------------------------------------------------------------------------------------------
struct FeedForward {
  bool f32, pair;   // types of the arrays; products of pairs
  const void *x, *wg, *wu, *wd, *gy;
  int64_t M;
  int C, H, act;
  int32_t *status;
  cudaStream_t st;
  const char *what;
};

// A caller's matrix: read where it lies, or laid out in the workspace by the job that is added.
static Matrix take_matrix(Carve &w, PrepArgs &prep, int64_t &blocks, const FeedForward &f, const void *src, int64_t rows, int cols) {
  if (!f.pair && cols % 8 == 0 && aligned16(src)) {
    Matrix m;
    m.at = static_cast<uint16_t *>(const_cast<void *>(src));
    m.rows = rows, m.cols = cols, m.ld = cols;
    return m;
  }
  const Matrix m = new_matrix(w, f.pair, rows, cols, 1);
  PrepJob &j = prep.job[prep.jobs++];
  j = PrepJob{src, m.at, f.pair ? m.at + m.plane() : nullptr, m.scale, rows, blocks, cols, (int)m.ld, (int)m.blocks_n(), !f.f32};
  blocks += m.blocks_m() * m.blocks_n();
  return m;
}
// Rows as pairs, brought to one size, the first of the launch's jobs; and as contributions to sums over rows.
struct TakenRows {
  Matrix x, gy, x_sum, gy_sum;
  float *s = nullptr, *t = nullptr;
};
static TakenRows take_rows(Carve &w, PrepArgs &prep, int64_t &blocks, const FeedForward &f, bool x_sum, bool gy_sum) {
  TakenRows r;
  RowsJob &j = prep.rows;
  const bool back = f.gy != nullptr;
  Matrix *const all[4] = {&r.x, &r.gy, &r.x_sum, &r.gy_sum};
  const bool wanted[4] = {true, back, x_sum, gy_sum};
  r.s = w.take<float>(up(f.M, 256));
  if (back) r.t = w.take<float>(up(f.M, 256));
  for (int o = 0; o < 4; o++)
    if (wanted[o]) {
      *all[o] = new_matrix(w, true, f.M, f.C, 1);
      j.hi[o] = reinterpret_cast<__half *>(all[o]->at), j.scale[o] = all[o]->scale;
    }
  j.src[0] = f.x, j.src[1] = f.gy, j.size[0] = r.s, j.size[1] = r.t, j.sources = back ? 2 : 1;
  j.rows = f.M, j.cols = f.C, j.plane = r.x.plane(), j.ld = (int)r.x.ld, j.blocks_n = (int)r.x.blocks_n(), j.bf16 = !f.f32;
  j.wide = f.f32 && f.C % 4 == 0 && aligned16(f.x) && (!back || aligned16(f.gy));
  j.blocks = r.x.blocks_m();
  if (j.blocks_n > 2) {   // sizes by a kernel of their own
    j.slab = (int)up(std::max(256, (f.C + PREP_SLABS - 1) / PREP_SLABS), 64), j.slabs = (f.C + j.slab - 1) / j.slab;
    for (int k = 0; k < j.sources; k++) j.most[k] = w.take<float>(j.slabs * f.M);
    j.blocks *= j.blocks_n * j.sources;
  }
  blocks += j.blocks;
  return r;
}
static int encode_all(std::initializer_list<Matrix *> all, bool bf16, const char *what) {
  for (Matrix *m : all)
    if (const int rc = encode_matrix(&m->map, *m, 64, 64, bf16, what)) return rc;
  return CMACE_OK;
}
static int set_hidden_out(TpArgs &g, const Matrix &m, int box_cols, bool bf16, const char *what) {
  g.out[0].use_map = 1;
  for (int p = 0; p < 3 && m.scale; p++) g.out_scale[p] = m.scale + (m.batches > 1 ? p : 0) * m.blocks_m() * m.blocks_n();
  g.out_scale_ld = m.blocks_n();
  return encode_matrix(&g.out[0].map, m, box_cols, 32, bf16, what);
}
// rows of a caller's array: by TMA where it can address them
static int set_user_out(TpArgs &g, void *ptr, bool f32, int64_t rows, int cols, const char *what, int which = 1) {
  TpOut &o = g.out[which];
  o.ptr = ptr;
  o.ld = cols;
  o.batch = rows * (int64_t)cols;
  g.out_bf16 = !f32;
  const int bytes = f32 ? 4 : 2;
  o.use_map = aligned16(ptr) && (int64_t)cols * bytes % 16 == 0;
  if (o.use_map) return encode_tile_map(&o.map, ptr, bytes, !f32, cols, rows, 1, cols, rows * (int64_t)cols, f32 ? 16 : 32, 32, what);
  return CMACE_OK;
}

static TpCost cost_of(const TpArgs &g, bool pair) {
  return {g.rows, g.cols, (g.kblocks[0] + (g.segments > 1 ? g.kblocks[1] : 0)) / g.splits + 1, (int64_t)g.batches * g.splits, pair};
}
template <int ACT>
static int launch_gated(const FeedForward &f, TpArgs &g) {
  const TpCost cost = cost_of(g, f.pair);
  const bool pairs = cost(2, 128, 256) < cost(1, 128, 256);
  if (f.pair) return pairs ? tp_launch<TP_GATED, true, 128, 2, ACT>(g, f.st, f.what) : tp_launch<TP_GATED, true, 128, 1, ACT>(g, f.st, f.what);
  return pairs ? tp_launch<TP_GATED, false, 128, 2, ACT>(g, f.st, f.what) : tp_launch<TP_GATED, false, 128, 1, ACT>(g, f.st, f.what);
}
template <int ACT>
static int launch_back(const FeedForward &f, TpArgs &g) {
  const TpCost cost = cost_of(g, f.pair);   // half of its blocks have two projections' columns, half one's
  if (f.pair)
    return cost(2, 64, 96) < cost(1, 64, 96) ? tp_launch<TP_BACK, true, 64, 2, ACT>(g, f.st, f.what) : tp_launch<TP_BACK, true, 64, 1, ACT>(g, f.st, f.what);
  return cost(2, 128, 192) < cost(1, 64, 96) ? tp_launch<TP_BACK, false, 128, 2, ACT>(g, f.st, f.what)
                                             : tp_launch<TP_BACK, false, 64, 1, ACT>(g, f.st, f.what);
}
static int launch_plain(bool pair, TpArgs &g, cudaStream_t st, const char *what) {
  const TpCost cost = cost_of(g, pair);
  const int64_t one = cost(1, 128, 128), two = cost(2, 128, 128);
  if (pair) return two < one ? tp_launch<TP_PLAIN, true, 128, 2>(g, st, what) : tp_launch<TP_PLAIN, true, 128, 1>(g, st, what);
  if (cost(2, 256, 256) < std::min(one, two)) return tp_launch<TP_PLAIN, false, 256, 2>(g, st, what);
  return two < one ? tp_launch<TP_PLAIN, false, 128, 2>(g, st, what) : tp_launch<TP_PLAIN, false, 128, 1>(g, st, what);
}

// Splits of a sum over the hidden columns for [M, C] results whose tiles leave SMs idle, by what the products cost and, for a second kernel, its
// launch and its traffic (3 600 bytes a cycle), `second` cycles more.  Forward, without and with, us: float32 64 rows, 512 and 4 096: 50, 30; 100 rows,
// 256 and 2 048: 30, 22; bf16 the same 21.8, 18.3 and 14.8, 16.2: from 10 000 and 15 000 cycles on.  Forward and backward, 64 rows: 140, 79;
// bf16 64, 47; but outside a graph a call with gradients is 90 of host whatever its kernels take, and another launch 4 more: from 30 000.
static int row_splits(bool pair, int64_t M, int C, int kblocks, int64_t second) {
  int best = 1;
  int64_t least = 0;
  for (int s = 1; s <= 32 && 2 * s <= kblocks; s *= 2) {
    const TpCost cost{M, C, kblocks / s + 1, s, pair};
    int64_t c = std::min(cost(1, 128, 128), cost(2, 128, 128));
    if (!pair) c = std::min(c, cost(2, 256, 256));
    if (s > 1) c += second + (s + 1) * M * C / 450;
    if (s == 1 || c < least) best = s, least = c;
  }
  return best;
}
// a product whose rows go to the caller's array, by way of the splits' sums where there are any
static int launch_rows(const FeedForward &f, TpArgs &g, void *out, int splits, float *partial) {
  if (splits == 1) {
    if (const int rc = set_user_out(g, out, f.f32, f.M, f.C, f.what)) return rc;
    return launch_plain(f.pair, g, f.st, f.what);
  }
  const int ld = (int)up(f.C, 4);
  g.splits = splits;
  g.out[1].use_map = 1;
  if (const int rc = encode_tile_map(&g.out[1].map, partial, 4, false, f.C, f.M, splits, ld, f.M * ld, 16, 32, f.what)) return rc;
  if (const int rc = launch_plain(f.pair, g, f.st, f.what)) return rc;
  const RowsSum r{partial, out, f.M, ld, f.C, splits, f.C % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (f.f32 ? 15 : 7)) == 0};
  const dim3 grid((unsigned)((f.M * ld / 4 + 255) / 256));
  if (f.f32) launch_dense(rows_sum_kernel<float>, grid, 256, f.st, r);
  else launch_dense(rows_sum_kernel<__nv_bfloat16>, grid, 256, f.st, r);
  return check_launch(f.what);
}

static int run_prep(const PrepArgs &p, int64_t blocks, cudaStream_t st, const char *what) {
  if (blocks == 0) return CMACE_OK;
  if (blocks >= (int64_t)1 << 31) return fail(CMACE_ERR_UNSUPPORTED, "%s: too many rows", what);
  if (p.rows.slabs)
    launch_dense(row_most_kernel, dim3((unsigned)((p.rows.rows + 63) / 64), (unsigned)p.rows.slabs, (unsigned)p.rows.sources), PREP_THREADS,
                   st, p.rows);
  const dim3 grid((unsigned)blocks);
  if (!p.rows.blocks) launch_dense(prep_kernel<PREP_COPY>, grid, prep_threads(PREP_COPY), st, p);
  else if (p.rows.slabs) launch_dense(prep_kernel<PREP_BLOCKS>, grid, prep_threads(PREP_BLOCKS), st, p);
  else if (p.rows.sources == 2) launch_dense(prep_kernel<PREP_BOTH>, grid, prep_threads(PREP_BOTH), st, p);
  else launch_dense(prep_kernel<PREP_WHOLE>, grid, prep_threads(PREP_WHOLE), st, p);
  return check_launch(what);
}

// Splits of the weight gradients' sum over M, by what a number costs in units of a block of 64 rows of one tile (0.3 to 0.5 us): rounds
// of tiles, a few blocks each for filling the ring and putting the sums down, the kernel that adds the splits and its traffic.
static int weight_splits(int64_t M, int C, int H) {
  const int64_t tiles = 3 * ((C + 127) / 128) * (int64_t)((H + 127) / 128), kb = blocks64(M);
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 64 && s <= kb; s++) {
    double cost = (double)((tiles * s + 147) / 148) * ((double)((kb + s - 1) / s) + 6.0);
    if (s > 1) cost += 10.0 + s * 3.0 * C * H * 6e-6;
    if (s == 1 || cost < least) best = s, least = cost;
  }
  return best;
}

template <typename T, int M, bool GATED, int ACT>
static int launch_few(FewArgs g, cudaStream_t st, const char *what) {
  const int blocks = (g.N + FEW_COLS - 1) / FEW_COLS;
  g.cluster = 1;
  while (g.cluster < 8 && 2 * g.cluster * blocks <= 148 && g.K >= 128 * g.cluster) g.cluster *= 2;
  constexpr int V = few_cols<T, M>();
  g.wide = g.N % V == 0;
  for (int i = 0; i < (GATED ? 2 : 1); i++) g.wide = g.wide && reinterpret_cast<uintptr_t>(g.w[i]) % (V * sizeof(T)) == 0;
  constexpr int SUMS = FEW_THREADS / 32 * (GATED ? 2 : 1) * FEW_COLS, SMEM = M * (FEW_K > SUMS ? FEW_K : SUMS) * 4;
  if (const int rc = allow_smem<few_rows_kernel<T, M, GATED, ACT>, SMEM>(what)) return rc;
  return launch_cluster(few_rows_kernel<T, M, GATED, ACT>, g.cluster, blocks * g.cluster, FEW_THREADS, SMEM, st, what, g);
}
template <typename T, int M, int ACT>
static int few_rows(const FeedForward &f, void *y, float *h) {
  FewArgs g{f.x, {f.wg, f.wu}, h, (int)f.M, f.C, f.H, 1, 0, f.status};
  if (const int rc = launch_few<T, M, true, ACT>(g, f.st, f.what)) return rc;
  g.x = h, g.w[0] = f.wd, g.out = y, g.K = f.H, g.N = f.C;
  return launch_few<T, M, false, ACT>(g, f.st, f.what);
}
template <typename T, int ACT>
static int few_rows(const FeedForward &f, void *y, float *h) {
  return f.M == 1 ? few_rows<T, 1, ACT>(f, y, h) : f.M == 2 ? few_rows<T, 2, ACT>(f, y, h) : f.M <= 4 ? few_rows<T, 4, ACT>(f, y, h) : few_rows<T, 8, ACT>(f, y, h);
}
template <typename T>
static int few_rows(const FeedForward &f, void *y, float *h) {
  return f.act == TP_SILU ? few_rows<T, TP_SILU>(f, y, h) : few_rows<T, TP_GELU>(f, y, h);
}

// CTAs of some_rows_kernel a block of rows: the hidden columns' groups are shared while SMs are free and every warp has one.
static int some_cluster(bool f32, int64_t M, int H) {
  const int64_t blocks = (M + SOME_ROWS - 1) / SOME_ROWS;
  const int groups = (H + some_group(f32) - 1) / some_group(f32);
  int cluster = 1;
  while (cluster < 8 && 2 * cluster * blocks <= 148 && groups > cluster * SOME_WARPS) cluster *= 2;
  return cluster;
}
template <typename T, int CT, int ACT>
static int launch_some(const FeedForward &f, void *y) {
  SomeArgs g{f.x, {f.wg, f.wu}, f.wd, y, f.M, f.C, f.H, 0, 1, 0};
  const int64_t blocks = (f.M + SOME_ROWS - 1) / SOME_ROWS;
  g.cluster = some_cluster(f.f32, f.M, f.H);
  // rows of x 64 (float32: quarters of a warp read two of them) or 32 bytes (halves read four) past a multiple of 128
  constexpr int SIZE = sizeof(T);
  g.ld = (int)(up(up(f.C, 16) * SIZE, 128) + (SIZE == 4 ? 64 : 32)) / SIZE;
  g.wide = f.H % (8 / SIZE) == 0 && f.C % 4 == 0 && ((reinterpret_cast<uintptr_t>(f.wg) | reinterpret_cast<uintptr_t>(f.wu)) & 7) == 0 &&
           ((reinterpret_cast<uintptr_t>(f.x) | reinterpret_cast<uintptr_t>(f.wd) | reinterpret_cast<uintptr_t>(y)) & (4 * SIZE - 1)) == 0;
  const int smem = (SIZE == 4 ? 2 : 1) * SOME_ROWS * g.ld * SIZE + SOME_WARPS * SOME_ROWS * 32 * CT * 4;
  constexpr int MOST = (SIZE == 4 ? 2 : 1) * SOME_ROWS * (32 * CT * SIZE + 128 + 64) + SOME_WARPS * SOME_ROWS * 32 * CT * 4;
  if (const int rc = allow_smem<some_rows_kernel<T, CT, ACT>, MOST>(f.what)) return rc;
  return launch_cluster(some_rows_kernel<T, CT, ACT>, g.cluster, blocks * g.cluster, SOME_THREADS, smem, f.st, f.what, g);
}
template <typename T, int ACT>
static int some_rows(const FeedForward &f, void *y) {
  return f.C <= 32 ? launch_some<T, 1, ACT>(f, y) : f.C <= 64 ? launch_some<T, 2, ACT>(f, y) : launch_some<T, 4, ACT>(f, y);
}
template <typename T>
static int some_rows(const FeedForward &f, void *y) {
  return f.act == TP_SILU ? some_rows<T, TP_SILU>(f, y) : some_rows<T, TP_GELU>(f, y);
}
// Whether the kernel above is the fastest, in ns of a recorded call, from lines through what was measured (up to 8 000 rows, widths
// 16 to 128, hidden widths 16 to 512; in brackets: this kernel and the others; us): float32, 100 rows: 32 and 64 (3.9, 12.2), 32 and 512
// (5.8, 15.9), 128 and 512 (12.0, 17.6), 100 and 301 (13.6, 17.6); 8 000 rows, 64 and 256: (40, 17).  bf16, 100 rows: 32 and 64 (3.4, 8.4), 128 and 512
// (8.9, 10.7), 33 and 70 (6.1, 13.1); 8 000 rows, 64 and 256 (19, 11).  One row, 128 and 512: float32 (11.2, 6.3), bf16 (8.5, 6.7).  Beyond
// 128 columns y takes the registers that the loads need: at 256 and 512, 22 against 19 in float32, 15 against 11 in bf16.
// Sizes alone decide, not addresses: the workspace is asked for without them.
static bool some_rows_pay(const FeedForward &f) {
  if (f.C > 128) return false;
  const int cluster = some_cluster(f.f32, f.M, f.H), group = some_group(f.f32);
  const int64_t each = ((f.H + group - 1) / group + cluster * SOME_WARPS - 1) / (cluster * SOME_WARPS);   // groups a warp
  const int64_t rounds = ((f.M + SOME_ROWS - 1) / SOME_ROWS * cluster + 147) / 148;
  const bool wide = f.C % 4 == 0 && f.H % (f.f32 ? 2 : 4) == 0, tma = f.f32 || (f.C % 8 == 0 && f.H % 8 == 0);
  const int64_t one = (f.f32 ? 53 : 34) * f.C * (wide ? 2 : f.f32 ? 3 : 6) / 2;   // a group
  const int64_t some = rounds * ((f.f32 ? 2800 : 2400) + each * one) + (cluster > 1 ? 1700 : 0);
  if (f.M <= FEW_ROWS) return f.H <= 1024 && some < 5600 + 300 * f.M + 15 * f.C + 2 * f.H;   // with 2 us of a second launch; long weights want all SMs
  const int64_t blocks = (f.C + 63) / 64 + (f.H + 63) / 64;
  return some < (f.f32 ? 10800 + 500 * blocks : (tma ? 8000 : 12000) + 200 * blocks);
}

static int forward(const FeedForward &f, void *y, Carve &w) {
  if (some_rows_pay(f)) return !w.base ? CMACE_OK : (f.f32 ? some_rows<float>(f, y) : some_rows<__nv_bfloat16>(f, y));
  if (f.M <= FEW_ROWS) {
    float *h = w.take<float>(f.M * f.H);
    return !w.base ? CMACE_OK : (f.f32 ? few_rows<float>(f, y, h) : few_rows<__nv_bfloat16>(f, y, h));
  }
  PrepArgs prep;
  memset(&prep, 0, sizeof(prep));
  int64_t blocks = 0;
  TakenRows rows;
  if (f.pair) rows = take_rows(w, prep, blocks, f, false, false);
  else rows.x = take_matrix(w, prep, blocks, f, f.x, f.M, f.C);
  Matrix &x = rows.x;
  Matrix wg = take_matrix(w, prep, blocks, f, f.wg, f.C, f.H);
  Matrix wu = take_matrix(w, prep, blocks, f, f.wu, f.C, f.H);
  Matrix wd = take_matrix(w, prep, blocks, f, f.wd, f.H, f.C);
  Matrix h = new_matrix(w, f.pair, f.M, f.H, 1);
  const int splits = row_splits(f.pair, f.M, f.C, blocks64(f.H), f.pair ? 10000 : 15000);
  float *partial = splits > 1 ? w.take<float>(splits * f.M * up(f.C, 4)) : nullptr;
  if (!w.base) return CMACE_OK;
  const bool bf16 = !f.pair;
  int rc = run_prep(prep, blocks, f.st, f.what);
  if (!rc) rc = encode_all({&x, &wg, &wu, &wd, &h}, bf16, f.what);
  TpArgs g = new_args(f.M, f.H, f.status);
  set_operand(g.a[0], x, true);
  set_operand(g.b[0], wg, false);
  set_operand(g.b[1], wu, false);
  set_k(g, 0, f.C);
  g.row_size[0] = rows.s;
  if (!rc) rc = set_hidden_out(g, h, 32, bf16, f.what);
  if (!rc) rc = f.act == TP_SILU ? launch_gated<TP_SILU>(f, g) : launch_gated<TP_GELU>(f, g);
  g = new_args(f.M, f.C, f.status);
  set_operand(g.a[0], h, true);
  set_operand(g.b[0], wd, false);
  set_k(g, 0, f.H);
  g.row_size[0] = g.row_size[1] = rows.s;
  if (!rc) rc = launch_rows(f, g, y, splits, partial);
  return rc;
}

static int backward(const FeedForward &f, void *gx, void *const gw[3], bool want_x, bool want_w, Carve &w) {
  PrepArgs prep;
  memset(&prep, 0, sizeof(prep));
  int64_t blocks = 0;
  TakenRows rows;
  const bool sum_x = want_w && (!w.base || gw[0] || gw[1]), sum_gy = want_w && (!w.base || gw[2]);   // when counting: room for both
  if (f.pair) {
    rows = take_rows(w, prep, blocks, f, sum_x, sum_gy);
  } else {
    rows.x_sum = rows.x = take_matrix(w, prep, blocks, f, f.x, f.M, f.C);
    rows.gy_sum = rows.gy = take_matrix(w, prep, blocks, f, f.gy, f.M, f.C);
  }
  Matrix &x = rows.x, &gy = rows.gy, &x_sum = rows.x_sum, &gy_sum = rows.gy_sum;
  Matrix wg = take_matrix(w, prep, blocks, f, f.wg, f.C, f.H);
  Matrix wu = take_matrix(w, prep, blocks, f, f.wu, f.C, f.H);
  Matrix wd = take_matrix(w, prep, blocks, f, f.wd, f.H, f.C);
  Matrix hidden = new_matrix(w, f.pair, f.M, f.H, 3);   // dg, du, h
  const int64_t ld = up(f.H, 4);
  const int splits = weight_splits(f.M, f.C, f.H);
  float *partial = want_w && splits > 1 ? w.take<float>((int64_t)splits * 3 * f.C * ld) : nullptr;
  const int x_splits = row_splits(f.pair, f.M, f.C, 2 * blocks64(f.H), 30000);
  float *x_partial = want_x && x_splits > 1 ? w.take<float>(x_splits * f.M * up(f.C, 4)) : nullptr;
  if (!w.base) return CMACE_OK;
  const bool bf16 = !f.pair;
  int rc = run_prep(prep, blocks, f.st, f.what);
  if (!rc) rc = encode_all({&x, &wg, &wu, &wd, &gy, &hidden}, bf16, f.what);
  if (f.pair) {
    if (!rc && sum_x) rc = encode_all({&x_sum}, bf16, f.what);
    if (!rc && sum_gy) rc = encode_all({&gy_sum}, bf16, f.what);
  } else {
    x_sum.map = x.map, gy_sum.map = gy.map;
  }
  TpArgs g = new_args(f.M, f.H, f.status);
  set_operand(g.a[0], x, true);
  set_operand(g.a[1], gy, true);
  set_operand(g.b[0], wg, false);
  set_operand(g.b[1], wu, false);
  set_operand(g.b[2], wd, true);
  g.segments = 2;
  set_k(g, 0, f.C);
  set_k(g, 1, f.C);
  g.row_size[0] = rows.s;
  if (!rc) rc = set_hidden_out(g, hidden, 16, bf16, f.what);
  if (!rc) rc = f.act == TP_SILU ? launch_back<TP_SILU>(f, g) : launch_back<TP_GELU>(f, g);
  if (want_x) {
    g = new_args(f.M, f.C, f.status);
    set_operand(g.a[0], hidden.part(0), true);
    set_operand(g.a[1], hidden.part(1), true);
    set_operand(g.b[0], wg, true);
    set_operand(g.b[1], wu, true);
    g.segments = 2;
    set_k(g, 0, f.H);
    set_k(g, 1, f.H);
    g.row_size[0] = rows.s, g.row_size[1] = rows.t;
    if (!rc) rc = launch_rows(f, g, gx, x_splits, x_partial);
  }
  if (want_w && splits == 1) {
    if (gw[0] || gw[1]) {
      g = new_args(f.C, f.H, f.status);
      set_operand(g.a[0], x_sum, false);
      set_operand(g.b[0], gw[0] && gw[1] ? hidden : hidden.part(gw[0] ? 0 : 1), false);
      g.batches = gw[0] && gw[1] ? 2 : 1;
      g.out_of_batch = 1;
      set_k(g, 0, f.M);
      if (!rc) rc = set_user_out(g, gw[0] ? gw[0] : gw[1], f.f32, f.C, f.H, f.what, 0);
      if (!rc && g.batches == 2) rc = set_user_out(g, gw[1], f.f32, f.C, f.H, f.what, 1);
      if (!rc) rc = launch_plain(f.pair, g, f.st, f.what);
    }
    if (gw[2]) {
      g = new_args(f.H, f.C, f.status);
      set_operand(g.a[0], hidden.part(2), false);
      set_operand(g.b[0], gy_sum, false);
      set_k(g, 0, f.M);
      if (!rc) rc = set_user_out(g, gw[2], f.f32, f.H, f.C, f.what);
      if (!rc) rc = launch_plain(f.pair, g, f.st, f.what);
    }
  } else if (want_w) {
    // batches dg, du and h: x^T dg, x^T du and, as its transpose, dy^T h
    g = new_args(f.C, f.H, f.status);
    set_operand(g.a[0], sum_x ? x_sum : gy_sum, false);   // one that is not wanted: any, its sums go nowhere
    set_operand(g.a[1], sum_gy ? gy_sum : x_sum, false);
    set_operand(g.b[0], hidden, false);
    g.batches = 3;
    g.splits = splits;
    g.a_of_last = 1;
    set_k(g, 0, f.M);
    g.out[1].use_map = 1;
    if (!rc) rc = encode_tile_map(&g.out[1].map, partial, 4, false, f.H, f.C, (int64_t)splits * 3, ld, (int64_t)f.C * ld, 16, 32, f.what);
    if (!rc) rc = launch_plain(f.pair, g, f.st, f.what);
    WeightReduce r{partial, {gw[0], gw[1], gw[2]}, ld, splits, f.C, f.H};
    const dim3 grid((unsigned)((f.H + 31) / 32), (unsigned)((f.C + 31) / 32), 3);
    if (!rc) {
      if (f.f32) launch_dense(weight_reduce_kernel<float>, grid, 256, f.st, r);
      else launch_dense(weight_reduce_kernel<__nv_bfloat16>, grid, 256, f.st, r);
      rc = check_launch(f.what);
    }
  }
  return rc;
}

// bf16 rounds h, dg and du once more, which makes 1.4 times the error of a result that is rounded alone: on the mean.  Where an array has few values,
// chance would make it more (128 hidden values, 300 of a gradient: 1.3 to 1.55), and all goes as pairs, like float32; that costs a kernel, 5 us.
static bool as_pairs(bool f32, int64_t M, int C, int H, bool backward) {
  return f32 || M * H <= 512 || M * C <= 1024 || (backward && (int64_t)C * H <= 1024);
}

static int check_sizes(const char *what, int64_t M, int C, int H, int act) {
  if (M < 0 || M > ((int64_t)1 << 31) - 1024 || C < 1 || H < 1) return fail(CMACE_ERR_ARG, "%s: bad sizes: %lld rows, width %d, hidden width %d", what, (long long)M, C, H);
  if (C > 1 << 20 || H > 1 << 20) return fail(CMACE_ERR_UNSUPPORTED, "%s: widths up to 2^20", what);
  if (act != TP_SILU && act != TP_GELU) return fail(CMACE_ERR_ARG, "%s: unknown activation %d", what, act);
  return CMACE_OK;
}

static int run_forward(bool f32, const void *x, const void *wg, const void *wu, const void *wd, int64_t M, int C, int H, int act, void *y,
                       void *workspace, int64_t bytes, int32_t *status, cmace_stream_t stream, const char *what) {
  if (int rc = check_sizes(what, M, C, H, act)) return rc;
  if (M == 0) return CMACE_OK;
  if (!x || !wg || !wu || !wd || !y || !workspace) return fail(CMACE_ERR_ARG, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(CMACE_ERR_ARG, "%s: the workspace has to be aligned to 256 bytes", what);
  FeedForward f{f32, as_pairs(f32, M, C, H, false), x, wg, wu, wd, nullptr, M, C, H, act, status, (cudaStream_t)stream, what};
  Carve count{nullptr};
  forward(f, y, count);
  count.used = std::max<int64_t>(count.used, 256);   // what is asked for at least
  if (bytes < count.used) return fail(CMACE_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what, (long long)bytes, (long long)count.used);
  ChainScope chain;
  chain_launches() = Chain::from_second;
  Carve w{static_cast<char *>(workspace)};
  return forward(f, y, w);
}

static int run_backward(bool f32, const void *x, const void *wg, const void *wu, const void *wd, const void *gy, int64_t M, int C, int H, int act,
                        void *gx, void *gwg, void *gwu, void *gwd, void *workspace, int64_t bytes, int32_t *status, cmace_stream_t stream,
                        const char *what) {
  if (int rc = check_sizes(what, M, C, H, act)) return rc;
  void *const gw[3] = {gwg, gwu, gwd};
  const bool want_w = gwg || gwu || gwd;
  const cudaStream_t st = (cudaStream_t)stream;
  if (M == 0) {   // a sum over no rows
    for (void *p : gw)
      if (p && cudaMemsetAsync(p, 0, (size_t)C * H * (f32 ? 4 : 2), st) != cudaSuccess) return check_launch(what);
    return CMACE_OK;
  }
  if (!gx && !want_w) return CMACE_OK;
  if (!x || !wg || !wu || !wd || !gy || !workspace) return fail(CMACE_ERR_ARG, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(CMACE_ERR_ARG, "%s: the workspace has to be aligned to 256 bytes", what);
  FeedForward f{f32, as_pairs(f32, M, C, H, true), x, wg, wu, wd, gy, M, C, H, act, status, st, what};
  Carve count{nullptr};
  backward(f, gx, gw, gx != nullptr, want_w, count);
  if (bytes < count.used) return fail(CMACE_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what, (long long)bytes, (long long)count.used);
  ChainScope chain;
  chain_launches() = Chain::from_second;
  Carve w{static_cast<char *>(workspace)};
  return backward(f, gx, gw, gx != nullptr, want_w, w);
}

}  // namespace cmace

using namespace cmace;

extern "C" {

int64_t cmace_dense_launches(void) { return dense_launches().load(std::memory_order_relaxed); }

int64_t cmace_gated_ff_workspace_bytes(int is_f32, int64_t rows, int width, int hidden, int backward_pass) {
  if (check_sizes("cmace_gated_ff_workspace_bytes", rows, width, hidden, TP_SILU)) return -1;
  if (rows == 0) return 256;
  // addresses are not known here: room for copies of all arrays of a width that is not a multiple of eight, and of those that are
  FeedForward f{is_f32 != 0, as_pairs(is_f32 != 0, rows, width, hidden, backward_pass != 0), (const void *)1, (const void *)1, (const void *)1, (const void *)1, backward_pass ? (const void *)1 : nullptr, rows, width, hidden, TP_SILU, nullptr, nullptr, ""};
  Carve count{nullptr};
  void *const none[3] = {nullptr, nullptr, nullptr};
  if (backward_pass) backward(f, nullptr, none, true, true, count);
  else forward(f, nullptr, count);
  return std::max<int64_t>(count.used, 256);
}

int cmace_gated_ff_fwd_f32(const float *x, const float *w_gate, const float *w_up, const float *w_down, int64_t rows, int width, int hidden,
                           int activation, float *y, void *workspace, int64_t workspace_bytes, int32_t *status, cmace_stream_t stream) {
  return run_forward(true, x, w_gate, w_up, w_down, rows, width, hidden, activation, y, workspace, workspace_bytes, status, stream,
                     "cmace_gated_ff_fwd_f32");
}
int cmace_gated_ff_fwd_bf16(const void *x, const void *w_gate, const void *w_up, const void *w_down, int64_t rows, int width, int hidden,
                            int activation, void *y, void *workspace, int64_t workspace_bytes, int32_t *status, cmace_stream_t stream) {
  return run_forward(false, x, w_gate, w_up, w_down, rows, width, hidden, activation, y, workspace, workspace_bytes, status, stream,
                     "cmace_gated_ff_fwd_bf16");
}
int cmace_gated_ff_bwd_f32(const float *x, const float *w_gate, const float *w_up, const float *w_down, const float *grad_y, int64_t rows, int width,
                           int hidden, int activation, float *grad_x, float *grad_gate, float *grad_up, float *grad_down, void *workspace,
                           int64_t workspace_bytes, int32_t *status, cmace_stream_t stream) {
  return run_backward(true, x, w_gate, w_up, w_down, grad_y, rows, width, hidden, activation, grad_x, grad_gate, grad_up, grad_down, workspace,
                      workspace_bytes, status, stream, "cmace_gated_ff_bwd_f32");
}
int cmace_gated_ff_bwd_bf16(const void *x, const void *w_gate, const void *w_up, const void *w_down, const void *grad_y, int64_t rows, int width,
                            int hidden, int activation, void *grad_x, void *grad_gate, void *grad_up, void *grad_down, void *workspace,
                            int64_t workspace_bytes, int32_t *status, cmace_stream_t stream) {
  return run_backward(false, x, w_gate, w_up, w_down, grad_y, rows, width, hidden, activation, grad_x, grad_gate, grad_up, grad_down, workspace,
                      workspace_bytes, status, stream, "cmace_gated_ff_bwd_bf16");
}

}  // extern "C"
