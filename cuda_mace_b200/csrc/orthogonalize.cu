// Newton-Schulz products that bring a stack of matrices near their orthogonal factors: X = U / (|U| + eps) (Frobenius norm), then `steps`
// times X <- a X + (b S + c S S) X with S = X X^T, or X <- a X + X (b S + c S S) with S = X^T X where that side is shorter.  A singular
// value s goes to a s + b s^3 + c s^5, so all of them meet near 1.
//
// What the precision asks for: a small singular value is multiplied by a up to `steps` times (485 with the usual coefficients), and so is
// what rounding adds along its direction.  X itself is therefore kept to 22 bits or more, as a pair of fp16 values (tile_product.cuh; 2^-50 of its bound
// where values are far below that), and
// a X formed from both; the operands of the products may be rounded further, since what that adds lies in the rows or in the columns of the large values, turns their
// vectors by the rounding and is not multiplied.  float32 takes pairs there too.  bf16 takes the high values alone (2^-12 instead of the
// result's 2^-9) but for S S, the smallest of the products, whose rounding weighs most: with pairs there the error of a result is 1.2 to
// 1.4 times that of its own rounding, without 1.6 to 1.8.  fp16's range suffices without looking at the values: |X|_2 <= 1 bounds every entry of X, S and b S + c S S in
// every step, and the host makes powers of two of the bounds (ns_step).
//
// Measured (B200, us a call of five steps, launches and all): one kernel: 4 of 64 x 64 20, 40 of 128 x 128 37, 3 of 128 x 512 in four CTAs each 59;
// a kernel a product: 1 of 1 001 x 250 154 (17 launches of 6 to 9: chains of first copies, four to 16 blocks of 64 k, an epilogue),
// 2 of 1 024 x 4 096 in bf16 320 (X X^T 20, S S 12, P X 28 a step; at 50 to 64 bytes a cycle and SM the copies of 128 x 256 operands
// take as long as their products).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "tile_product.cuh"

namespace cmace {

constexpr int NS_THREADS = 256;
constexpr int NS_CHUNKS = 512;   // partial sums of a matrix at most

// ---- the powers of two of a step ----------------------------------------------------------------------------------------------
// Largest |t (a + b t^2 + c t^4)| over [0, most], from its ends and the zeros of its derivative
__host__ __device__ inline double most_odd(double a, double b, double c, double most) {
  const auto at = [=](double t) { return fabs(t * (a + t * t * (b + t * t * c))); };
  double best = at(most);
  // a + 3 b q + 5 c q^2 = 0, q = t^2
  if (c != 0) {
    const double d = 9 * b * b - 20 * a * c;
    if (d >= 0)
      for (int k = -1; k <= 1; k += 2) {
        const double q = (-3 * b + k * sqrt(d)) / (10 * c);
        if (q > 0 && q < most * most) best = fmax(best, at(sqrt(q)));
      }
  } else if (b != 0 && -a / (3 * b) > 0 && -a / (3 * b) < most * most) {
    best = fmax(best, at(sqrt(-a / (3 * b))));
  }
  return best;
}
// largest |t (b + c t)|
__host__ __device__ inline double most_square(double b, double c, double most) {
  const auto at = [=](double t) { return fabs(t * (b + t * c)); };
  const double best = at(most);
  return c != 0 && -b / (2 * c) > 0 && -b / (2 * c) < most ? fmax(best, at(-b / (2 * c))) : best;
}
// The power of two above `most` and 5 % more, for what rounding adds
__host__ __device__ inline int exponent_of(double most) {
  int e = 0;
  if (most != 0) frexp(most * 1.05, &e);   // most * 1.05 < 2^e
  return e;
}
// keeps values up to `most` below 2^15.  What is below 2^-45 of the other values may be lost: products of scales stay float32 values.
__host__ __device__ inline float fp16_scale(double most) {
  const int e = exponent_of(most);
  return (float)ldexp(1.0, 15 - (e > -45 ? e : -45));
}
// One step on X^ = X 2^-k, whose singular values (those of X up to `most`) are below 1, to X'^ = X' 2^-k':
// X'^ = a 2^(k-k') X^ + P^ X^ with P^ = b 2^(3k-k') S^ + c 2^(5k-k') S^ S^.  So the values of every step are of one size however far the polynomial
// shrinks X or lets it grow, and the last step brings 2^k' back.
struct alignas(32) NsStep {
  float a, b, c, ss, sp, out, unused[2];   // ss, sp: powers of two of the pairs of S^ and P^; out: of what the step leaves
};
constexpr float NS_SX = 0x1p15f;   // of the pairs of X^
constexpr int NS_MAX_STEPS = 100;
// most, k: of the step, then of the next one
__host__ __device__ inline NsStep ns_step(double a, double b, double c, bool last, double &most, int &k) {
  const double next = most_odd(a, b, c, most), size = ldexp(most, -k), size_s = size * size;
  const int to = exponent_of(next);
  const double b_k = ldexp(b, 3 * k - to), c_k = ldexp(c, 5 * k - to);
  const NsStep s = {(float)ldexp(a, k - to), (float)b_k, (float)c_k, fp16_scale(size_s), fp16_scale(most_square(b_k, c_k, size_s)),
                    last ? (float)ldexp(1.0, to) : 1.f, {0.f, 0.f}};
  most = next, k = to;
  return s;
}

struct NsPrep {
  const void *src;
  double *partial;   // [count][chunks]
  __half *h;         // [count][hi, lo][rows][ld]
  int64_t count, rows;
  int cols, ld, chunks, bf16, blocks;   // blocks of ns_prep_kernel a matrix
  double eps;
  double a, b, c;
  int steps;
  NsStep *own;       // [count][NS_MAX_STEPS]: of a matrix far smaller than eps, whose X begins far below the bound of 1; ss = 0: the call's
};

__device__ __forceinline__ float ns_load(const void *p, int64_t i, int bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]) : static_cast<const float *>(p)[i];
}
// values i .. i + n - 1 (n <= 8) of an array; wide: i is a multiple of eight of an array aligned to 16 bytes, and all eight are there
__device__ __forceinline__ void ns_load8(float (&v)[8], const void *p, int64_t i, int n, int bf16, bool wide) {
  if (!wide) {
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = k < n ? ns_load(p, i + k, bf16) : 0.f;
  } else if (bf16) {
    const uint4 x = __ldg(reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(p) + i));
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 4; k++) v[2 * k] = __uint_as_float(w[k] << 16), v[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
  } else {
    const float4 *f = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
    const float4 x = __ldg(f), y = __ldg(f + 1);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
  }
}

// size / (|U| + eps) as two factors, the first a power of two: |U| of a matrix of float32's largest or smallest values leaves float32's range.
struct NsInverse {
  float first, second;
  __device__ __forceinline__ NsInverse(double square, double eps, double size = 1.0) {
    const double inv = size / (sqrt(square) + eps);
    first = inv > 0x1p100 ? 0x1p100f : inv < 0x1p-100 ? 0x1p-100f : 1.0f;
    second = (float)(inv / first);
  }
  __device__ __forceinline__ float operator*(float v) const { return v * first * second; }
};

// Squares of eight values in float32 where those neither leave its range nor fall below it, in float64 otherwise and from there on: neither
// large nor small updates are lost, and the sum of a matrix is one value whatever its size.
__global__ void __launch_bounds__(NS_THREADS) ns_norm_kernel(const NsPrep p) {
  __shared__ double sums[NS_THREADS / 32];
  grid_begin();
  const int64_t n = p.rows * p.cols, m = blockIdx.x / (unsigned)p.chunks, c = blockIdx.x - m * p.chunks, n8 = (n + 7) / 8;
  const int64_t i0 = n8 * c / p.chunks, i1 = n8 * (c + 1) / p.chunks;
  const bool wide = n % 8 == 0 && (reinterpret_cast<uintptr_t>(p.src) & 15) == 0;
  double s = 0;
#pragma unroll 4
  for (int64_t i = i0 + threadIdx.x; i < i1; i += NS_THREADS) {
    float v[8], t = 0.f;
    ns_load8(v, p.src, m * n + 8 * i, (int)min((int64_t)8, n - 8 * i), p.bf16, wide);
#pragma unroll
    for (int k = 0; k < 8; k++) t = fmaf(v[k], v[k], t);
    if (t > 1e-30f && t < 1e30f) {
      s += t;
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++) s = fma((double)v[k], (double)v[k], s);
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < NS_THREADS / 32; w++) s += sums[w];
    p.partial[blockIdx.x] = s;
  }
}

// X of the first step as pairs; a thread takes eight columns of a row, four times.  Where |U| is far below eps, X begins far below 1, and the
// bounds with it: the matrix has steps of its own.
__global__ void __launch_bounds__(NS_THREADS) ns_prep_kernel(const NsPrep p) {
  grid_begin();
  const int64_t m = blockIdx.x / (unsigned)p.blocks, b = blockIdx.x - m * p.blocks;
  double s = 0;   // every warp sums the partial sums, in the same order
  for (int c = threadIdx.x & 31; c < p.chunks; c += 32) s += __ldcg(p.partial + m * p.chunks + c);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  double most = sqrt(s) / (sqrt(s) + p.eps);
  const bool small = most < 0.25 && most > 0;
  int k = exponent_of(small ? most : 1.0);
  const NsInverse inv(s, p.eps, ldexp((double)NS_SX, -k));
  if (b == 0 && threadIdx.x == 0)
    for (int i = 0; i < p.steps; i++) {
      NsStep own = {};
      if (small) own = ns_step(p.a, p.b, p.c, i + 1 == p.steps, most, k);
      p.own[m * NS_MAX_STEPS + i] = own;
    }
  const int per_row = (p.cols + 7) / 8;
  const int64_t items = p.rows * per_row, plane = p.rows * p.ld;
  const bool wide = p.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(p.src) & 15) == 0;
  __half *hi = p.h + m * 2 * plane;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int64_t item = (b * 4 + i) * NS_THREADS + threadIdx.x;
    if (item >= items) break;
    const int64_t row = item / per_row;
    const int col = (int)(item - row * per_row) * 8;
    float v[8];
    ns_load8(v, p.src, (m * p.rows + row) * p.cols + col, p.cols - col < 8 ? p.cols - col : 8, p.bf16, wide);
    uint32_t h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; k++) tp_split2(inv * v[2 * k], inv * v[2 * k + 1], 1.f, h[k], l[k]);
    __half *to = hi + row * p.ld + col;   // rows have a multiple of 64 elements
    *reinterpret_cast<uint4 *>(to) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4 *>(to + plane) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

// ---- all steps in one kernel, for matrices whose shorter side fits a tile ------------------------------------------------------
// X [side <= 128, columns] (a tall matrix is read and written transposed) stays on the SM: as fp16 pairs in shared memory, which
// serve S = X X^T (contracted index inside a row) and P X (contracted index over the rows) from the same image, and in float32 in
// tensor memory.  S, then P = b S + c S S, go the same way.  A matrix of more than 128 columns is spread over the CTAs of a cluster: each
// has its columns of X and a part of S; every CTA adds up the parts' rows that are its own, in the order of the ranks, and hands their pairs
// to all.  (A stack that fills the SMs keeps up to 256 columns in one CTA.)
//
// The three products of a step and what stands between them form a chain, so the block works on one thing at a time: 16 warps for the
// elementwise phases (a warp of each quarter of the lanes has a quarter of the columns), one thread issues MMAs.  Terms with a low part come
// first: the sum is small while they are added, and the truncating additions that count are the 4 a 64 k of hi hi.
//
// A_TMEM (up to 128 columns a CTA): the A operands are in tensor memory too, since an MMA of 128 columns with both operands in shared
// memory takes 85 to 100 cycles instead of 64.  Columns: sum 128, X 128, hi and lo of S or P 128, of X 128.  With 256 columns: sum, X.
constexpr int NSF_THREADS = 512;
constexpr int NSF_STAGE_LD = 65;          // floats a row of the transposing buffer
constexpr int NSF_IMAGE = 128 * 128;      // 128 rows of 64 fp16
constexpr int NSF_S_BYTES = 4 * NSF_IMAGE;   // two chunks, hi and lo

struct NsFused {
  const void *src;
  void *out;
  int64_t count;
  int side, length, tall, bf16, steps, columns, chunks;   // columns of a CTA, its chunks of 64
  int cluster;
  double eps;
  int32_t *status;
  NsStep step[NS_MAX_STEPS];
};

__device__ __forceinline__ void peer_store2(uint32_t addr, uint32_t x, uint32_t y) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ float4 peer_load4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void smem_store4(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 smem_load4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// D = A B + D 2^-11, A in tensor memory
__device__ __forceinline__ void umma_f16_ts_low(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, 11;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc)
      : "memory");
}
// two packed fp16 of each part as the floats that they stand for, times their power of two
__device__ __forceinline__ float2 pair_value(uint32_t hi, uint32_t lo) {
  const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&hi)), y = __half22float2(*reinterpret_cast<const __half2 *>(&lo));
  return make_float2(fmaf(y.x, 0x1p-11f, x.x), fmaf(y.y, 0x1p-11f, x.y));
}
// WORDS packed values of one row (16-byte pieces `piece`, ... of its 128 bytes) into an image
template <int WORDS>
__device__ __forceinline__ void put_row(uint32_t image, int row, int piece, const uint32_t (&w)[WORDS]) {
#pragma unroll
  for (int c = 0; c < WORDS / 4; c++) smem_store4(image + (uint32_t)sw128_offset(row, piece + c), w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
}
template <int N>
__device__ __forceinline__ void split_row(const float (&v)[N], float scale, uint32_t (&hi)[N / 2], uint32_t (&lo)[N / 2]) {
#pragma unroll
  for (int k = 0; k < N / 2; k++) tp_split2(v[2 * k], v[2 * k + 1], scale, hi[k], lo[k]);
}

template <int CLUSTER, bool A_TMEM>
__global__ void __launch_bounds__(NSF_THREADS, 1) ns_fused_kernel(const __grid_constant__ NsFused g) {
  static_assert(CLUSTER == 1 || A_TMEM, "up to 128 columns a CTA of a cluster");
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t done_bar, peer_bars[2];
  __shared__ uint32_t tmem_base_slot;
  __shared__ double sums[NSF_THREADS / 32 + 1];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char *const generic = smem_raw + (base - raw);
  const uint32_t x_hi = base, x_lo = base + (uint32_t)(g.chunks * NSF_IMAGE), s_hi = base + (uint32_t)(2 * g.chunks * NSF_IMAGE);
  const uint32_t s_lo = s_hi + 2 * NSF_IMAGE, part = s_hi + NSF_S_BYTES;   // part: this CTA's part of S
  float *const stage = reinterpret_cast<float *>(generic + (s_hi - base));   // before and after the steps
  const uint32_t bar = smem_u32(&done_bar);
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31, q = warp & 3, group = warp >> 2;
  const int row = 32 * q + lane;
  const uint32_t rank = CLUSTER > 1 ? cluster_rank() : 0;

  if (tid == 0) {
    mbar_init(bar, 1);
    mbar_init(smem_u32(&peer_bars[0]), CLUSTER);
    mbar_init(smem_u32(&peer_bars[1]), CLUSTER);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tmem_alloc(smem_u32(&tmem_base_slot), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)uniform((int)tmem_base_slot);
  const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16), master = acc + (A_TMEM ? 128 : 256);
  const uint32_t s_tmem = acc + 256, x_tmem = acc + 384;   // A_TMEM: hi in 64 columns, lo in the next 64
  grid_begin();
  const int64_t matrix = blockIdx.x / (unsigned)CLUSTER;
  const int64_t size = (int64_t)g.side * g.length;
  const int col0 = (int)rank * g.columns;
  uint32_t phase = 0;
  bool ok = true;

  // ---- the update into tensor memory, and its norm -----------------------------------------------------------------------
  double square = 0;
  constexpr int AHEAD = A_TMEM ? 2 : 1;   // chunks on their way at once
  float v[AHEAD][16];
  // a thread's 16 values of a chunk: of one column and every eighth row, or (tall) of one row and every fourth column
  struct Mine {
    int64_t first, step;
    int n;   // of them in the matrix
  };
  const auto mine_of = [&](int ch) {
    Mine m;
    const int r0 = g.tall ? tid & 127 : tid >> 6, in = 64 * ch + (g.tall ? tid >> 7 : tid & 63), end = min(g.columns, g.length - col0);
    m.n = g.tall ? (r0 < g.side ? (end - in + 3) / 4 : 0) : (in < end ? (g.side - r0 + 7) / 8 : 0);
    m.first = matrix * size + (g.tall ? (int64_t)(col0 + in) * g.side + r0 : (int64_t)r0 * g.length + col0 + in);
    m.step = g.tall ? 4 * (int64_t)g.side : 8 * (int64_t)g.length;
    return m;
  };
  const auto fetch = [&](int ch, float (&to)[16]) {
    const Mine m = mine_of(ch);
    if (g.bf16) {
      const __nv_bfloat16 *from = static_cast<const __nv_bfloat16 *>(g.src) + m.first;
#pragma unroll
      for (int k = 0; k < 16; k++, from += m.step) to[k] = k < m.n ? __bfloat162float(*from) : 0.f;
    } else {
      const float *from = static_cast<const float *>(g.src) + m.first;
#pragma unroll
      for (int k = 0; k < 16; k++, from += m.step) to[k] = k < m.n ? *from : 0.f;
    }
  };
#pragma unroll
  for (int a = 0; a < AHEAD; a++)
    if (a < g.chunks) fetch(a, v[a]);
  for (int first = 0; first < g.chunks; first += AHEAD) {
#pragma unroll
    for (int a = 0; a < AHEAD; a++) {
      const int ch = first + a;
      if (ch >= g.chunks) break;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 16; k++) {
        const int e = tid + NSF_THREADS * k;
        stage[g.tall ? (e & 127) * NSF_STAGE_LD + (e >> 7) : (e >> 6) * NSF_STAGE_LD + (e & 63)] = v[a][k];
        square = fma((double)v[a][k], (double)v[a][k], square);
      }
      if (ch + AHEAD < g.chunks) fetch(ch + AHEAD, v[a]);
      __syncthreads();
      uint32_t w[16];
#pragma unroll
      for (int k = 0; k < 16; k++) w[k] = __float_as_uint(stage[row * NSF_STAGE_LD + 16 * group + k]);
      tmem_st16(master + (uint32_t)(64 * ch + 16 * group), w);
    }
  }
  tmem_st_wait();
  // sums in the same order everywhere: of a warp's lanes, of the warps, of the CTAs of a cluster
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) square += __shfl_xor_sync(0xffffffffu, square, d);
  if (lane == 0) sums[warp] = square;
  __syncthreads();
  square = sums[lane & 15];
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) square += __shfl_xor_sync(0xffffffffu, square, d);
  if (CLUSTER > 1) {
    if (tid == 0) sums[NSF_THREADS / 32] = square;
    cluster_sync();
    square = 0;
#pragma unroll
    for (int r = 0; r < CLUSTER; r++) {
      double other;
      asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(other) : "r"(peer_smem(smem_u32(&sums[NSF_THREADS / 32]), (uint32_t)r)) : "memory");
      square += other;
    }
  }
  const NsInverse inv(square, g.eps);
  // a chunk's pairs of X: shared memory, and tensor memory where it has room
  const auto put_x = [&](int ch, const float (&x)[16], float scale) {
    uint32_t hi[8], lo[8];
    split_row(x, scale, hi, lo);
    put_row(x_hi + (uint32_t)(ch * NSF_IMAGE), row, 2 * group, hi);
    put_row(x_lo + (uint32_t)(ch * NSF_IMAGE), row, 2 * group, lo);
    if (A_TMEM) {
      tmem_st8(x_tmem + (uint32_t)(32 * ch + 8 * group), hi);
      tmem_st8(x_tmem + (uint32_t)(64 + 32 * ch + 8 * group), lo);
    }
  };
  for (int ch = 0; ch < g.chunks; ch++) {
    const uint32_t at = master + (uint32_t)(64 * ch + 16 * group);
    uint32_t w[16];
    float x[16];
    tmem_ld16_nowait(at, w);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 16; k++) x[k] = 0.5f * (inv * __uint_as_float(w[k]));   // |X| <= 1: the first k is 1
#pragma unroll
    for (int k = 0; k < 16; k++) w[k] = __float_as_uint(x[k]);
    tmem_st16(at, w);
    put_x(ch, x, NS_SX);
  }
  tmem_st_wait();

  const int side16 = (g.side + 15) & ~15;
  const uint32_t idesc_s = tp_idesc(side16, 0, 0, 0), idesc_x = tp_idesc(64 * g.chunks, 0, 0, 1);
  // Operands are written, sums are read: products of A and B over `steps16` times 16 k, three terms, the ones with a low part first.
  // Descriptors of an image's steps differ by constants: one thread issues all MMAs, at some ten cycles an instruction.
  const uint64_t lo_of_x = (uint64_t)(g.chunks * (NSF_IMAGE >> 4)), lo_of_s = 2 * (NSF_IMAGE >> 4);
  const uint64_t x_desc = tp_desc(x_hi, 0), s_desc = tp_desc(s_hi, 0);
  // X with its rows as k: runs of 64 columns an image apart
  const uint64_t x_rows = (tp_desc(x_hi, 1) & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(NSF_IMAGE >> 4) << 16);
  const auto products = [&](uint32_t a_tmem, uint64_t A, uint64_t a_lo, uint64_t B, uint64_t b_lo, int steps16, auto b_mn, uint32_t idesc) {
    constexpr bool B_MN = decltype(b_mn)::value;
    constexpr int MOST = B_MN || A_TMEM ? 8 : 16;   // 128 rows, 128 or 256 columns
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    if (warp == 0 && elect_one()) {
      tc_fence_after();
      const auto product = [&](int k, uint64_t al, uint64_t bl, uint32_t accumulate) {
        const uint64_t b = B + bl + (uint64_t)(B_MN ? k * 128 : (k >> 2) * (NSF_IMAGE >> 4) + (k & 3) * 2);
        if (A_TMEM) umma_f16_ts(tmem, a_tmem + (uint32_t)(8 * k) + (al ? 64u : 0u), b, idesc, accumulate);
        else umma_16(tmem, A + al + (uint64_t)((k >> 2) * (NSF_IMAGE >> 4) + (k & 3) * 2), b, idesc, accumulate);
      };
      // the terms with a low part, which is kept times 2^11, then the first of the others on 2^-11 of their sum
#pragma unroll
      for (int k = 0; k < MOST; k++) {
        if (k >= steps16) break;
        product(k, a_lo, 0, k > 0);
        product(k, 0, b_lo, 1);
      }
      if (A_TMEM) umma_f16_ts_low(tmem, a_tmem, B, idesc);
      else umma_16_low(tmem, A, B, idesc);
#pragma unroll
      for (int k = 1; k < MOST; k++) {
        if (k >= steps16) break;
        product(k, 0, 0, 1);
      }
      umma_commit(bar);
    }
    if (ok && !warp_wait(bar, phase, lane)) {   // a block that gave up goes on: the others of its cluster meet it at the barriers
      if (lane == 0 && g.status) atomicCAS(g.status, 0, 107);
      ok = false;
    }
    phase ^= 1;
    tc_fence_after();
  };
  const uint32_t s_first = tmem + 256, x_first = tmem + 384;   // lane 0 of the A operands
  const int s_piece = 4 * (group & 1);                          // this thread's 32 columns of S
  const uint32_t s_at = (uint32_t)((group >> 1) * NSF_IMAGE);
  const bool mine = 32 * group < side16;   // columns from side16 on are not written by a product, and none reads what is made of them
  const int x_steps = (min(g.columns, g.length - col0 > 0 ? g.length - col0 : 1) + 15) / 16;

  uint32_t peer_phase = 0;
  const auto meet = [&](int which) {
    const uint32_t peer_bar = smem_u32(&peer_bars[which]);
    __syncthreads();
    if (tid < CLUSTER) peer_arrive(peer_bar, (uint32_t)tid);
    if (ok && !peer_wait(peer_bar, peer_phase)) {
      if (lane == 0 && g.status) atomicCAS(g.status, 0, 110);
      ok = false;
    }
  };
  for (int step = 0; step < g.steps; step++) {
    const NsStep &now = g.step[step];
    const float ss = now.ss, sp = now.sp;
    uint32_t u[32] = {}, hi[16] = {}, lo[16] = {};
    float s[32];
    // S = X X^T
    products(x_first, x_desc, lo_of_x, x_desc, lo_of_x, x_steps, std::false_type{}, idesc_s);
    if (mine) tmem_ld32(acc + (uint32_t)(32 * group), u);
    const float to_s = 1.0f / (NS_SX * NS_SX);
#pragma unroll
    for (int j = 0; j < 32; j++) s[j] = __uint_as_float(u[j]) * to_s;
    if (CLUSTER == 1) {
      if (mine) {
        split_row(s, ss, hi, lo);
        put_row(s_hi + s_at, row, s_piece, hi);
        put_row(s_lo + s_at, row, s_piece, lo);
      }
    } else {
      // part: [128 rows][32 pieces of four columns], the piece changed by the row: a warp's accesses meet all banks.  Between SMs it is bytes
      // that count, 11 to 12 a cycle here whichever side moves them: each CTA fetches its share of the rows and sends pairs.
      if (mine)
#pragma unroll
        for (int c = 0; c < 8; c++)
          smem_store4(part + (uint32_t)(row * 512 + (((8 * group + c) ^ (row & 31)) << 4)), __float_as_uint(s[4 * c]), __float_as_uint(s[4 * c + 1]),
                      __float_as_uint(s[4 * c + 2]), __float_as_uint(s[4 * c + 3]));
      meet(0);
      // four columns a lane: a warp's loads are a row of up to 512 bytes on end
      const int share = (side16 + CLUSTER - 1) / CLUSTER, piece = lane;
#pragma unroll 2
      for (int r = (int)rank * share + warp; r < min((int)(rank + 1) * share, side16); r += NSF_THREADS / 32) {
        if (4 * piece >= side16) break;
        const uint32_t from = part + (uint32_t)(r * 512 + ((piece ^ (r & 31)) << 4));
        float4 x[CLUSTER];
#pragma unroll
        for (int p = 0; p < CLUSTER; p++) x[p] = peer_load4(peer_smem(from, (uint32_t)p));
        float sum[4] = {};
#pragma unroll
        for (int p = 0; p < CLUSTER; p++) sum[0] += x[p].x, sum[1] += x[p].y, sum[2] += x[p].z, sum[3] += x[p].w;
        uint32_t h[2], l[2];
        split_row(sum, ss, h, l);
        const uint32_t to = (uint32_t)((piece >> 4) * NSF_IMAGE + sw128_offset(r, (piece & 15) >> 1) + (piece & 1) * 8);
#pragma unroll
        for (int p = 0; p < CLUSTER; p++) {
          peer_store2(peer_smem(s_hi + to, (uint32_t)p), h[0], h[1]);
          peer_store2(peer_smem(s_lo + to, (uint32_t)p), l[0], l[1]);
        }
      }
      meet(1);   // products() fences the images for the tensor cores
      peer_phase ^= 1;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const uint32_t at = s_at + (uint32_t)sw128_offset(row, s_piece + c);
        const uint4 h = smem_load4(s_hi + at), l = smem_load4(s_lo + at);
        hi[4 * c] = h.x, hi[4 * c + 1] = h.y, hi[4 * c + 2] = h.z, hi[4 * c + 3] = h.w;
        lo[4 * c] = l.x, lo[4 * c + 1] = l.y, lo[4 * c + 2] = l.z, lo[4 * c + 3] = l.w;
      }
      const float from = 1.0f / ss;
#pragma unroll
      for (int k = 0; k < 16; k++) {
        const float2 x = pair_value(hi[k], lo[k]);
        s[2 * k] = x.x * from, s[2 * k + 1] = x.y * from;
      }
    }
    if (A_TMEM) {
      tmem_st16(s_tmem + (uint32_t)(16 * group), hi);
      tmem_st16(s_tmem + (uint32_t)(64 + 16 * group), lo);
      tmem_st_wait();
    }
    // P = b S + c S S
    products(s_first, s_desc, lo_of_s, s_desc, lo_of_s, side16 / 16, std::false_type{}, idesc_s);
    if (mine) {
      tmem_ld32(acc + (uint32_t)(32 * group), u);
      const float from_ss = now.c / (ss * ss);
#pragma unroll
      for (int j = 0; j < 32; j++) s[j] = now.b * s[j] + from_ss * __uint_as_float(u[j]);
      split_row(s, sp, hi, lo);
      if (!A_TMEM) {
        put_row(s_hi + s_at, row, s_piece, hi);
        put_row(s_lo + s_at, row, s_piece, lo);
      }
    }
    if (A_TMEM) {
      tmem_st16(s_tmem + (uint32_t)(16 * group), hi);
      tmem_st16(s_tmem + (uint32_t)(64 + 16 * group), lo);
      tmem_st_wait();
    }
    // X = a X + P X
    products(s_first, s_desc, lo_of_s, x_rows, lo_of_x, side16 / 16, std::true_type{}, idesc_x);
    const float from_p = now.out / (sp * NS_SX), from_x = now.a * now.out;
    const bool last = step + 1 == g.steps;
#pragma unroll(A_TMEM ? 2 : 1)
    for (int ch = 0; ch < g.chunks; ch++) {
      const uint32_t col = (uint32_t)(64 * ch + 16 * group);
      uint32_t w[16], m[16];
      float x[16];
      tmem_ld16_nowait(acc + col, w);
      tmem_ld16_nowait(master + col, m);
      tmem_ld_wait();
#pragma unroll
      for (int k = 0; k < 16; k++) x[k] = from_x * __uint_as_float(m[k]) + from_p * __uint_as_float(w[k]);
      if (!last) {
#pragma unroll
        for (int k = 0; k < 16; k++) m[k] = __float_as_uint(x[k]);
        tmem_st16(master + col, m);
        put_x(ch, x, NS_SX);
      } else {
        __syncthreads();   // every warp has its sums: the image of S is free; and the stores of the chunk before are done
#pragma unroll
        for (int k = 0; k < 16; k++) stage[row * NSF_STAGE_LD + 16 * group + k] = x[k];
        __syncthreads();
        const Mine m = mine_of(ch);
        const float *from = stage + (g.tall ? (tid & 127) * NSF_STAGE_LD + (tid >> 7) : (tid >> 6) * NSF_STAGE_LD + (tid & 63));
        const int next = g.tall ? 4 : 8 * NSF_STAGE_LD;
        if (g.bf16) {
          __nv_bfloat16 *to = static_cast<__nv_bfloat16 *>(g.out) + m.first;
#pragma unroll
          for (int k = 0; k < 16; k++, to += m.step)
            if (k < m.n) *to = __float2bfloat16_rn(from[k * next]);
        } else {
          float *to = static_cast<float *>(g.out) + m.first;
#pragma unroll
          for (int k = 0; k < 16; k++, to += m.step)
            if (k < m.n) *to = from[k * next];
        }
      }
    }
    tmem_st_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (CLUSTER > 1) {   // nobody reads or writes a block's shared memory after it has left
    __syncwarp();
    cluster_sync();
  }
  if (warp == 0) tmem_dealloc(tmem, 512);
}

struct NsCall {
  bool f32;
  const void *src;
  void *out;
  int64_t count, rows;
  int cols, steps;
  double a, b, c, eps;
  int32_t *status;
  cudaStream_t st;
  const char *what;
};

struct NsVariant {
  int ctas, tn;
};
static NsVariant ns_variant(bool pair, int64_t rows, int cols, int kblocks, int64_t count) {
  const TpCost cost{rows, cols, kblocks, count, pair};
  const int64_t one = cost(1, 128, 128), two = cost(2, 128, 128);
  if (!pair && cost(2, 256, 256) < std::min(one, two)) return {2, 256};
  return {two < one ? 2 : 1, 128};
}
template <int KIND>
static int launch_ns(NsVariant v, TpArgs &g, cudaStream_t st, const char *what) {
  return v.ctas == 2 ? tp_launch<KIND, true, 128, 2>(g, st, what) : tp_launch<KIND, true, 128, 1>(g, st, what);
}
template <int KIND>
static int launch_ns_single(NsVariant v, TpArgs &g, cudaStream_t st, const char *what) {
  if (v.tn == 256) return tp_launch<KIND, false, 256, 2>(g, st, what);
  return v.ctas == 2 ? tp_launch<KIND, false, 128, 2>(g, st, what) : tp_launch<KIND, false, 128, 1>(g, st, what);
}

// CTAs a matrix for the kernel above, 0: it does not fit
static int fused_cluster(int64_t count, int64_t rows, int cols) {
  const int64_t side = std::min<int64_t>(rows, cols), length = std::max<int64_t>(rows, cols);
  if (side > 128 || length > 1024) return 0;
  // one of 128 x 160: 44 us in one CTA, 49 in two; of 128 x 256: 53 and 51 (64 x 160: 33 and 35, 64 x 256: 39 and 35)
  if (length <= 192 || (length <= 256 && count > 74)) return 1;
  int p = 2;
  while (p * 128 < length) p *= 2;
  return p;
}

constexpr int fused_smem(int cluster, int chunks) { return 2 * chunks * NSF_IMAGE + NSF_S_BYTES + (cluster > 1 ? 128 * 512 : 0) + 1024; }
template <int CLUSTER, bool A_TMEM>
static int launch_fused(const NsCall &f, const NsFused &g, int smem) {
  constexpr int MOST = fused_smem(CLUSTER, A_TMEM ? 2 : 4);
  if (const int rc = allow_smem<ns_fused_kernel<CLUSTER, A_TMEM>, MOST>(f.what)) return rc;
  return launch_cluster(ns_fused_kernel<CLUSTER, A_TMEM>, CLUSTER, f.count * CLUSTER, NSF_THREADS, smem, f.st, f.what, g);
}

static int run_fused(const NsCall &f, int cluster) {
  NsFused g;
  memset(&g, 0, sizeof(g));
  g.src = f.src, g.out = f.out, g.count = f.count;
  g.tall = f.rows > f.cols;
  g.side = (int)std::min<int64_t>(f.rows, f.cols), g.length = (int)std::max<int64_t>(f.rows, f.cols);
  g.bf16 = !f.f32, g.steps = f.steps, g.cluster = cluster;
  g.columns = (int)up((g.length + cluster - 1) / cluster, 16);
  g.chunks = (g.columns + 63) / 64;
  g.eps = f.eps, g.status = f.status;
  double most = 1.0;
  int k = exponent_of(most);
  for (int i = 0; i < f.steps; i++) g.step[i] = ns_step(f.a, f.b, f.c, i + 1 == f.steps, most, k);
  const int smem = fused_smem(cluster, g.chunks);
  switch (cluster) {
    case 2: return launch_fused<2, true>(f, g, smem);
    case 4: return launch_fused<4, true>(f, g, smem);
    case 8: return launch_fused<8, true>(f, g, smem);
    default: return g.chunks <= 2 ? launch_fused<1, true>(f, g, smem) : launch_fused<1, false>(f, g, smem);
  }
}
// how far singular values can grow is what fp16 operands and float32 sums have to hold
static int check_growth(const NsCall &f) {
  double most = 1.0;
  for (int k = 0; k < f.steps; k++) {
    const double p = most_square(f.b, f.c, most * most), next = most_odd(f.a, f.b, f.c, most);
    if (!(next < 1e12) || !(p < 1e12))
      return fail(CMACE_ERR_ARG, "%s: coefficients %g, %g, %g: singular values may grow to %g in step %d", f.what, f.a, f.b, f.c, next, k + 1);
    most = next;
  }
  return CMACE_OK;
}

static int orthogonalize(const NsCall &f, Carve &w) {
  if (const int cluster = fused_cluster(f.count, f.rows, f.cols)) return w.base ? run_fused(f, cluster) : CMACE_OK;
  const bool wide = f.rows <= f.cols;   // S = X X^T, else X^T X
  const int side = wide ? (int)f.rows : f.cols;
  const int64_t n = f.rows * f.cols;
  const int chunks = (int)std::min<int64_t>(NS_CHUNKS, (n + 8191) / 8192);
  double *partial = w.take<double>(f.count * chunks);
  NsStep *own = w.take<NsStep>(f.count * NS_MAX_STEPS);
  Matrix x[2];
  for (Matrix &m : x) m = new_matrix(w, true, f.rows, f.cols, f.count, 64, false);
  Matrix s = new_matrix(w, true, side, side, f.count, 64, false), poly = new_matrix(w, true, side, side, f.count, 64, false);
  if (!w.base) return CMACE_OK;

  double most = 1.0;   // bound of the singular values
  int k = exponent_of(most);
  const int blocks = (int)((f.rows * ((f.cols + 7) / 8) + 4 * NS_THREADS - 1) / (4 * NS_THREADS));
  NsPrep p{f.src, partial, reinterpret_cast<__half *>(x[0].at), f.count, f.rows, f.cols, (int)x[0].ld, chunks, f.f32 ? 0 : 1, blocks, f.eps, f.a, f.b, f.c, f.steps, own};
  launch_dense(ns_norm_kernel, dim3((unsigned)(f.count * chunks)), NS_THREADS, f.st, p);
  launch_dense(ns_prep_kernel, dim3((unsigned)(f.count * blocks)), NS_THREADS, f.st, p);
  int rc = check_launch(f.what);
  // maps: operands; what is added and written, in boxes of the variants' columns a warp
  const int kb_s = blocks64(wide ? f.cols : f.rows), kb = blocks64(side);
  const NsVariant v_gram = ns_variant(f.f32, side, side, kb_s, f.count), v_poly = ns_variant(true, side, side, kb, f.count),
                  v_apply = ns_variant(f.f32, f.rows, f.cols, kb, f.count);
  CUtensorMap part_x[2], to_s, from_s, to_poly;
  TpOut to_out;
  memset(&to_out, 0, sizeof(to_out));
  for (Matrix *m : {&x[0], &x[1], &s, &poly})
    if (!rc) rc = encode_matrix(&m->map, *m, 64, 64, false, f.what);
  for (int k = 0; k < 2 && !rc; k++) rc = encode_matrix(&part_x[k], x[k], v_apply.tn / 4, 32, false, f.what);
  if (!rc) rc = encode_matrix(&to_s, s, v_gram.tn / 4, 32, false, f.what);
  if (!rc) rc = encode_matrix(&from_s, s, v_poly.tn / 4, 32, false, f.what);
  if (!rc) rc = encode_matrix(&to_poly, poly, v_poly.tn / 4, 32, false, f.what);
  const int bytes = f.f32 ? 4 : 2;
  to_out.ptr = f.out, to_out.ld = f.cols, to_out.batch = n;
  to_out.use_map = aligned16(f.out) && (int64_t)f.cols * bytes % 16 == 0;
  if (!rc && to_out.use_map) rc = encode_tile_map(&to_out.map, f.out, bytes, !f.f32, f.cols, f.rows, f.count, f.cols, n, 16, 32, f.what);

  for (int step = 0; step < f.steps && !rc; step++) {
    const Matrix &now = x[step & 1];
    const bool last = step + 1 == f.steps;
    const NsStep by = ns_step(f.a, f.b, f.c, last, most, k);
    TpArgs g = new_args(side, side, f.status);
    g.batches = (int)f.count;
    g.in_f16 = 1;
    g.own = reinterpret_cast<const float4 *>(own + step), g.own_stride = NS_MAX_STEPS * (int)(sizeof(NsStep) / sizeof(float4));
    set_k(g, 0, wide ? f.cols : f.rows);
    set_operand(g.a[0], now, wide);
    set_operand(g.b[0], now, wide);
    g.out[0].map = to_s;
    g.alpha = 1.0f / (NS_SX * NS_SX);
    g.pair_scale = by.ss;
    rc = f.f32 ? launch_ns<TP_GRAM>(v_gram, g, f.st, f.what) : launch_ns_single<TP_GRAM>(v_gram, g, f.st, f.what);

    set_k(g, 0, side);
    set_operand(g.a[0], s, true);
    set_operand(g.b[0], s, true);
    g.out[0].map = to_poly;
    g.cin = from_s;
    g.alpha = by.c / (by.ss * by.ss), g.beta = by.b / by.ss, g.pair_scale = by.sp;
    if (!rc) rc = launch_ns<TP_POLY>(v_poly, g, f.st, f.what);

    g.rows = f.rows, g.cols = f.cols;
    set_operand(g.a[0], wide ? poly : now, true);
    set_operand(g.b[0], wide ? now : poly, !wide);
    g.out[0].map = part_x[(step + 1) & 1];
    g.out[1] = to_out;
    g.out_bf16 = !f.f32;
    g.cin = part_x[step & 1];
    g.alpha = by.out / (by.sp * NS_SX), g.beta = by.a * by.out / NS_SX, g.pair_scale = last ? 0.f : NS_SX;
    if (!rc) rc = f.f32 ? launch_ns<TP_APPLY>(v_apply, g, f.st, f.what) : launch_ns_single<TP_APPLY>(v_apply, g, f.st, f.what);
  }
  return rc;
}

static int check_ns(const char *what, int64_t count, int64_t rows, int cols, int steps) {
  if (count < 0 || rows < 1 || cols < 1 || steps < 1 || steps > 100)
    return fail(CMACE_ERR_ARG, "%s: bad sizes: %lld matrices of %lld x %d, %d steps", what, (long long)count, (long long)rows, cols, steps);
  if (rows > 1 << 20 || cols > 1 << 20 || count * ((rows + 31) / 32) * ((cols + 31) / 32) >= (int64_t)1 << 30)
    return fail(CMACE_ERR_UNSUPPORTED, "%s: sides up to 2^20 and fewer than 2^30 blocks of 32 x 32", what);
  return CMACE_OK;
}

static int run_orthogonalize(bool f32, const void *update, int64_t count, int64_t rows, int cols, int steps, double a, double b, double c, double eps,
                             void *out, void *workspace, int64_t bytes, int32_t *status, cmace_stream_t stream, const char *what) {
  if (int rc = check_ns(what, count, rows, cols, steps)) return rc;
  if (count == 0) return CMACE_OK;
  if (!update || !out || !workspace) return fail(CMACE_ERR_ARG, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(CMACE_ERR_ARG, "%s: the workspace has to be aligned to 256 bytes", what);
  if (!(std::isfinite(a) && std::isfinite(b) && std::isfinite(c)) || !(eps >= 0)) return fail(CMACE_ERR_ARG, "%s: bad coefficients or eps", what);
  NsCall f{f32, update, out, count, rows, cols, steps, a, b, c, eps, status, (cudaStream_t)stream, what};
  if (const int rc = check_growth(f)) return rc;
  Carve need{nullptr};
  orthogonalize(f, need);
  if (bytes < need.used) return fail(CMACE_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what, (long long)bytes, (long long)need.used);
  ChainScope chain;
  chain_launches() = Chain::from_second;
  Carve w{static_cast<char *>(workspace)};
  return orthogonalize(f, w);
}

}  // namespace cmace

using namespace cmace;

extern "C" {

int64_t cmace_orthogonalize_workspace_bytes(int is_f32, int64_t count, int64_t rows, int cols) {
  if (check_ns("cmace_orthogonalize_workspace_bytes", count, rows, cols, 1)) return -1;
  NsCall f{is_f32 != 0, nullptr, nullptr, count, rows, cols, 1, 0, 0, 0, 0, nullptr, nullptr, ""};
  Carve need{nullptr};
  orthogonalize(f, need);
  return std::max<int64_t>(need.used, 256);
}
int cmace_orthogonalize_f32(const float *update, int64_t count, int64_t rows, int cols, int steps, double a, double b, double c, double eps, float *out,
                            void *workspace, int64_t workspace_bytes, int32_t *status, cmace_stream_t stream) {
  return run_orthogonalize(true, update, count, rows, cols, steps, a, b, c, eps, out, workspace, workspace_bytes, status, stream,
                           "cmace_orthogonalize_f32");
}
int cmace_orthogonalize_bf16(const void *update, int64_t count, int64_t rows, int cols, int steps, double a, double b, double c, double eps, void *out,
                             void *workspace, int64_t workspace_bytes, int32_t *status, cmace_stream_t stream) {
  return run_orthogonalize(false, update, count, rows, cols, steps, a, b, c, eps, out, workspace, workspace_bytes, status, stream,
                           "cmace_orthogonalize_bf16");
}

}  // extern "C"
