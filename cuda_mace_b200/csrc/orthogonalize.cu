// Newton-Schulz products that bring a stack of matrices near their orthogonal factors: X = U / (|U| + eps) (Frobenius norm), then `steps`
// times X <- a X + (b S + c S S) X with S = X X^T, or X <- a X + X (b S + c S S) with S = X^T X where that side is shorter.  A singular
// value s goes to a s + b s^3 + c s^5, so all of them meet near 1.
//
// What the precision asks for: a small singular value is multiplied by a up to `steps` times (485 with the usual coefficients), and so is
// what rounding adds along its direction.  X itself is therefore kept in float32 and a X formed from that; the operands of the
// products may be rounded further, since what that adds lies in the rows or in the columns of the large values, turns their
// vectors by the rounding and is not multiplied.  float32 takes pairs of fp16 values (tile_product.cuh), bf16 single fp16 values (2^-12 instead of
// the result's 2^-9).  fp16's range suffices without looking at the values: |X|_2 <= 1 bounds every entry of X, S and b S + c S S in
// every step, and the host makes powers of two of the bounds.
#include <algorithm>
#include <cmath>

#include "tile_product.cuh"

namespace cmace {

constexpr int NS_THREADS = 256;
constexpr int NS_CHUNKS = 64;   // partial sums of a matrix at most

struct NsPrep {
  const void *src;
  double *partial;   // [count][chunks]
  float *x;          // [count][rows][ld]
  __half *hi, *lo;   // [count][rows][ld]
  int64_t count, rows;
  int cols, ld, chunks, bf16;
  double eps;
  float scale;
};

__device__ __forceinline__ float ns_load(const void *p, int64_t i, int bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]) : static_cast<const float *>(p)[i];
}

// Squares in float64: neither large nor small updates leave the range, and the sum of a matrix is one value whatever its size.
__global__ void __launch_bounds__(NS_THREADS) ns_norm_kernel(const NsPrep p) {
  __shared__ double sums[NS_THREADS / 32];
  grid_begin();
  const int64_t n = p.rows * p.cols, m = blockIdx.x / p.chunks, c = blockIdx.x - m * p.chunks;
  const int64_t i0 = n * c / p.chunks, i1 = n * (c + 1) / p.chunks;
  double s = 0;
  for (int64_t i = i0 + threadIdx.x; i < i1; i += NS_THREADS) {
    const double v = ns_load(p.src, m * n + i, p.bf16);
    s = fma(v, v, s);
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

// A block of 32 rows x 32 columns of a matrix a CTA of 256 threads.
__global__ void __launch_bounds__(NS_THREADS) ns_prep_kernel(const NsPrep p) {
  grid_begin();
  const int64_t per = (p.rows + 31) / 32 * ((p.cols + 31) / 32);
  const int64_t m = blockIdx.x / per, b = blockIdx.x - m * per;
  const int nb = (p.cols + 31) / 32;
  const int64_t row0 = b / nb * 32;
  const int col = (int)(b - b / nb * nb) * 32 + (threadIdx.x & 31);
  double s = 0;
  for (int c = 0; c < p.chunks; c++) s += __ldcg(p.partial + m * p.chunks + c);
  const float inv = (float)(1.0 / (sqrt(s) + p.eps));
  if (col >= p.cols) return;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int64_t row = row0 + (threadIdx.x >> 5) + 8 * i;
    if (row >= p.rows) break;
    const float v = ns_load(p.src, (m * p.rows + row) * p.cols + col, p.bf16) * inv;
    const int64_t at = (m * p.rows + row) * p.ld + col;
    p.x[at] = v;
    if (p.lo) {
      uint32_t h, l;
      tp_split2(v * p.scale, 0.f, h, l);
      p.hi[at] = __ushort_as_half((unsigned short)h);
      p.lo[at] = __ushort_as_half((unsigned short)l);
    } else {
      p.hi[at] = __float2half_rn(v * p.scale);
    }
  }
}

// largest |p| over [0, most] of a polynomial c1 t + c3 t^3 + c5 t^5 (odd) or c1 t + c2 t^2, from its ends and the zeros of its derivative
static double most_odd(double a, double b, double c, double most) {
  const auto at = [&](double t) { return std::fabs(t * (a + t * t * (b + t * t * c))); };
  double best = at(most);
  // a + 3 b q + 5 c q^2 = 0, q = t^2
  if (c != 0) {
    const double d = 9 * b * b - 20 * a * c;
    if (d >= 0)
      for (double sign : {-1.0, 1.0}) {
        const double q = (-3 * b + sign * std::sqrt(d)) / (10 * c);
        if (q > 0 && q < most * most) best = std::max(best, at(std::sqrt(q)));
      }
  } else if (b != 0 && -a / (3 * b) > 0 && -a / (3 * b) < most * most) {
    best = std::max(best, at(std::sqrt(-a / (3 * b))));
  }
  return best;
}
static double most_square(double b, double c, double most) {
  const auto at = [&](double t) { return std::fabs(t * (b + t * c)); };
  double best = at(most);
  if (c != 0 && -b / (2 * c) > 0 && -b / (2 * c) < most) best = std::max(best, at(-b / (2 * c)));
  return best;
}
// power of two that keeps values up to `most`, and 5 % more for what rounding adds, below 2^15
static float fp16_scale(double most) {
  if (most == 0) return 1.f;
  int e;
  std::frexp(most * 1.05, &e);   // most * 1.05 < 2^e
  return (float)std::ldexp(1.0, 15 - e);
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

static int set_split_out(TpArgs &g, const Matrix &m, const char *what) {
  const void *base[2] = {m.hi, m.lo};
  for (int t = 0; t < (m.lo ? 2 : 1); t++) {
    const int rc = encode_tile_map(&g.out[t].map, base[t], 2, false, m.cols, m.rows, m.batches, m.ld, m.rows * m.ld, 32, 32, what);
    if (rc) return rc;
    g.out[t].use_map = 1;
  }
  return CMACE_OK;
}
template <int KIND>
static int launch_ns(bool pair, int tn, TpArgs &g, cudaStream_t st, const char *what) {
  if (tn == 256) return pair ? tp_launch<KIND, true, 256>(g, st, what) : tp_launch<KIND, false, 256>(g, st, what);
  return pair ? tp_launch<KIND, true, 128>(g, st, what) : tp_launch<KIND, false, 128>(g, st, what);
}

static int orthogonalize(const NsCall &f, Carve &w) {
  const bool wide = f.rows <= f.cols;   // S = X X^T, else X^T X
  const int side = wide ? (int)f.rows : f.cols;
  const int64_t n = f.rows * f.cols;
  const int chunks = (int)std::min<int64_t>(NS_CHUNKS, (n + 8191) / 8192);
  double *partial = w.take<double>(f.count * chunks);
  Matrix x[2];
  for (Matrix &m : x) m = new_matrix(w, f.f32, f.rows, f.cols, f.count, 64, false);
  const Matrix s = new_matrix(w, f.f32, side, side, f.count, 64, false), poly = new_matrix(w, f.f32, side, side, f.count, 64, false);
  float *master = w.take<float>(f.count * f.rows * x[0].ld);
  if (!w.base) return CMACE_OK;

  double most = 1.0;   // bound of the singular values
  float sx = fp16_scale(most);
  NsPrep p{f.src, partial, master, static_cast<__half *>(x[0].hi), static_cast<__half *>(x[0].lo), f.count, f.rows, f.cols, (int)x[0].ld, chunks,
           f.f32 ? 0 : 1, f.eps, sx};
  launch_chained(ns_norm_kernel, dim3((unsigned)(f.count * chunks)), dim3(NS_THREADS), (size_t)0, f.st, p);
  launch_chained(ns_prep_kernel, dim3((unsigned)(f.count * ((f.rows + 31) / 32) * ((f.cols + 31) / 32))), dim3(NS_THREADS), (size_t)0, f.st, p);
  int rc = check_launch(f.what);
  const int t_s = tile_columns(side, side, f.count), t_x = tile_columns(f.rows, f.cols, f.count);
  for (int step = 0; step < f.steps && !rc; step++) {
    const Matrix &now = x[step & 1], &next = x[(step + 1) & 1];
    const double most_s = most * most, most_p = most_square(f.b, f.c, most_s), most_next = most_odd(f.a, f.b, f.c, most);
    if (!(most_next < 1e12) || !(most_p < 1e12))
      return fail(CMACE_ERR_ARG, "%s: coefficients %g, %g, %g: singular values may grow to %g in step %d", f.what, f.a, f.b, f.c, most_next, step + 1);
    const float ss = fp16_scale(most_s), sp = fp16_scale(most_p), sn = fp16_scale(most_next);
    const bool last = step + 1 == f.steps;
    TpArgs g = new_args(side, side, f.status);
    g.batches = (int)f.count;
    g.in_f16 = 1;
    g.kblocks[0] = blocks64(wide ? f.cols : f.rows);
    if (!rc) rc = set_operand(g.a[0], now, wide, 128, false, f.what);
    if (!rc) rc = set_operand(g.b[0], now, wide, t_s, false, f.what);
    if (!rc) rc = set_split_out(g, s, f.what);
    g.alpha = 1.0f / (sx * sx);
    g.pair_scale = ss;
    if (!rc) rc = launch_ns<TP_GRAM>(f.f32, t_s, g, f.st, f.what);

    g.kblocks[0] = blocks64(side);
    if (!rc) rc = set_operand(g.a[0], s, true, 128, false, f.what);
    if (!rc) rc = set_operand(g.b[0], s, true, t_s, false, f.what);
    if (!rc) rc = set_split_out(g, poly, f.what);
    g.cin[0] = s.hi, g.cin[1] = s.lo, g.cin_ld = s.ld, g.cin_batch = side * s.ld;
    g.alpha = (float)f.c / (ss * ss), g.beta = (float)f.b / ss, g.pair_scale = sp;
    if (!rc) rc = launch_ns<TP_POLY>(f.f32, t_s, g, f.st, f.what);

    g.rows = f.rows, g.cols = f.cols;
    if (wide) {
      if (!rc) rc = set_operand(g.a[0], poly, true, 128, false, f.what);
      if (!rc) rc = set_operand(g.b[0], now, false, 64, false, f.what);
    } else {
      if (!rc) rc = set_operand(g.a[0], now, true, 128, false, f.what);
      if (!rc) rc = set_operand(g.b[0], poly, true, t_x, false, f.what);
    }
    if (!rc) rc = set_split_out(g, next, f.what);
    g.cin[0] = master, g.cin_ld = now.ld, g.cin_batch = f.rows * now.ld;
    g.alpha = 1.0f / (sp * sx), g.beta = (float)f.a, g.pair_scale = last ? 0.f : sn;
    TpOut &o = g.out[2];
    if (last) {
      const int bytes = f.f32 ? 4 : 2;
      o.ptr = f.out, o.ld = f.cols, o.batch = n;
      o.use_map = aligned16(f.out) && (int64_t)f.cols * bytes % 16 == 0;
      g.out_bf16 = !f.f32;
      if (!rc && o.use_map) rc = encode_tile_map(&o.map, f.out, bytes, !f.f32, f.cols, f.rows, f.count, f.cols, n, 32, 32, f.what);
    } else {
      o.use_map = 1;
      if (!rc) rc = encode_tile_map(&o.map, master, 4, false, f.cols, f.rows, f.count, now.ld, f.rows * now.ld, 32, 32, f.what);
    }
    if (!rc) rc = launch_ns<TP_APPLY>(f.f32, t_x, g, f.st, f.what);
    most = most_next;
    sx = sn;
  }
  return rc;
}

static int check_ns(const char *what, int64_t count, int64_t rows, int cols, int steps) {
  if (count < 0 || rows < 1 || cols < 1 || steps < 1 || steps > 100)
    return fail(CMACE_ERR_ARG, "%s: bad sizes: %lld matrices of %lld x %d, %d steps", what, (long long)count, (long long)rows, cols, steps);
  if (rows > 1 << 20 || cols > 1 << 20 || count * ((rows + 31) / 32) * ((cols + 31) / 32) >= (int64_t)1 << 31)
    return fail(CMACE_ERR_UNSUPPORTED, "%s: sides up to 2^20 and 2^31 blocks of 32 x 32", what);
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
