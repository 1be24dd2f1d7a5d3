// Orthogonalised updates by Newton-Schulz products, and the optimiser step around them.
//
//   X_0 = U / (|U|_F + eps)          (U transposed where it has more rows than columns, so that X is m x n with m <= n)
//   G = X X^T,  P = b G + c G G,  X <- a X + P X          once per coefficient triple (a, b, c)
// which moves every singular value of X towards 1 by the odd polynomial a s + b s^3 + c s^5 and leaves the singular vectors.
//   step:  buf <- mu buf + grad,  U = grad + mu buf (or buf),  W <- (1 - lr wd) W - lr sqrt(max(1, rows / cols)) X
//
// Bound by the matrix cores: per triple m^2 n + m^3 + 2 m^2 n operations, the two symmetric products at half (one triangle of tiles,
// each written twice).  X, G and P are held as two bf16 planes, about 17 bits (tile_gemm.h): in one plane the rounding of X
// pollutes the directions of small singular values, which the polynomial then multiplies by up to a^5 = 485 (relative error of
// the result 2e-2 on Gaussian updates, against 3e-5 with two planes; the result is rounded to bf16, 2e-3).
// The squared norm is summed in 64 bits: it neither overflows nor depends on how the update is cut.
#include "../../include/sgpo_hip.h"
#include "tile_gemm.h"

namespace {

constexpr int PARTS = 64;   // partial sums of a matrix's squared norm

__host__ __device__ inline int64_t round_up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

template <typename T> __device__ __forceinline__ float up(T v);
template <> __device__ __forceinline__ float up<float>(float v) { return v; }
template <> __device__ __forceinline__ float up<bf16_t>(bf16_t v) { return bf2f(v); }

struct Source {
  const void* grad;
  float* buf;              // null: the update is grad itself
  float momentum;
  int nesterov;
  int64_t stride_b, ld;    // of grad; buf is contiguous
  int rows, cols;
};

template <typename T>
__device__ __forceinline__ float update_at(const Source& s, int b, int r, int c) {   // after the buffer's own update
  const float g = up<T>(reinterpret_cast<const T*>(s.grad)[b * s.stride_b + r * s.ld + c]);
  if (!s.buf) return g;
  const float m = s.buf[((int64_t)b * s.rows + r) * s.cols + c];
  return s.nesterov ? fmaf(s.momentum, m, g) : m;
}

// momentum buffer, and partial sums of the update's squares
template <typename T>
__global__ __launch_bounds__(256) void square_kernel(Source s, double* part) {
  const int b = blockIdx.y;
  const int64_t total = (int64_t)s.rows * s.cols;
  double sum = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)PARTS * 256) {
    const int r = (int)(i / s.cols), c = (int)(i - (int64_t)r * s.cols);
    if (s.buf) {
      float* m = s.buf + (int64_t)b * total + i;
      *m = fmaf(s.momentum, *m, up<T>(reinterpret_cast<const T*>(s.grad)[b * s.stride_b + r * s.ld + c]));
    }
    const double u = (double)update_at<T>(s, b, r, c);
    sum += u * u;
  }
  __shared__ double share[4];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) share[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) part[b * PARTS + blockIdx.x] = share[0] + share[1] + share[2] + share[3];
}

__device__ __forceinline__ float inverse_norm(const double* part, double eps) {   // every lane of the wave calls it
  double s = part[threadIdx.x & 63];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  return (float)(1.0 / (sqrt(s) + eps));
}

// X [m][n] planes of the scaled update, zero in the padding columns; TALL: X is the update transposed
template <typename T, bool TALL>
__global__ __launch_bounds__(256) void load_kernel(Source s, const double* part, double eps, bf16_t* X, int m, int n, int64_t ldx, int64_t bstride) {
  __shared__ float tile[64][65];
  const int b = blockIdx.z, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  const float inv = inverse_norm(part + b * PARTS, eps);
  if constexpr (TALL) {
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
      const int c = i >> 6, r = i & 63;   // along the update's rows
      if (r0 + r < m && c0 + c < n) tile[r][c] = update_at<T>(s, b, c0 + c, r0 + r);
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 64 * 16; i += 256) {
    const int r = r0 + (i >> 4), c = c0 + (i & 15) * 4;
    if (r >= m || c >= ldx / 2) continue;
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = c + q < n ? inv * (TALL ? tile[r - r0][c - c0 + q] : update_at<T>(s, b, r, c + q)) : 0.f;
    tg::store4<2>(X + b * bstride + r * ldx, c, v);
  }
}

struct Mats {
  bf16_t *X, *Y, *G, *P;   // planes
  int64_t ldx, ldg, sx, sg;   // row pitch and batch stride, stored elements
  int m, n;
};

// tile (i, j), i <= j, of the triangle, row by row
__device__ __forceinline__ void triangle(int t, int tiles, int& i, int& j) {
  i = 0;
  while (t >= tiles - i) { t -= tiles - i; ++i; }
  j = i + t;
}

// G = X X^T (POLY false)  or  P = b G + c G G (POLY true): one triangle of tiles, each also written transposed
template <class S, bool POLY>
__global__ __launch_bounds__(S::THREADS, 2) void symmetric_kernel(Mats q, int tiles, float cb, float cc) {
  static_assert(S::BM == S::BN && S::PL == 2, "square tiles of two planes");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int i, j;
  triangle(blockIdx.x, tiles, i, j);
  const int b = blockIdx.y, m0 = i * S::BM, n0 = j * S::BN;
  const bf16_t* src = POLY ? q.G + b * q.sg : q.X + b * q.sx;
  const int64_t ld = POLY ? q.ldg : q.ldx;
  tg::Operand o{src, ld, q.m, 0};
  f32x4 acc[S::MT][S::NT];
  tg::clear<S>(acc);
  tg::run<S, tg::KC, tg::KC>(o, o, m0, n0, 0, (int)(ld / 64), smem, acc);
  bf16_t* dst = (POLY ? q.P : q.G) + b * q.sg;
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = (int)threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
  for (int x = 0; x < S::MT; ++x) {
    const int m = m0 + (wm * S::MT + x) * 16 + l16;
#pragma unroll
    for (int y = 0; y < S::NT; ++y) {
      const int n = n0 + (wn * S::NT + y) * 16 + 4 * l4;
      float v[4] = {acc[x][y][0], acc[x][y][1], acc[x][y][2], acc[x][y][3]};
      if (m < q.m && n < q.ldg / 2) {
        if constexpr (POLY) {
          float g[4];
          tg::load4<2>(q.G + b * q.sg + m * q.ldg, n, g);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = fmaf(cb, g[e], cc * v[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) if (n + e >= q.m) v[e] = 0.f;
        tg::store4<2>(dst + m * q.ldg, n, v);
      }
      if (i != j && m < q.ldg / 2) {   // the mirror image: row n + e, column m
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < q.m) {
            float pl[2];
            tg::split<2>(m < q.m ? v[e] : 0.f, pl);
            bf16_t* at = dst + (n + e) * q.ldg + (m >> 5) * 64 + (m & 31);
            at[0] = f2bf(pl[0]);
            at[32] = f2bf(pl[1]);
          }
      }
    }
  }
}

struct Result {
  void* out;               // bf16 [batch][rows][cols], or the weight
  int out_bf16;
  int tall, rows, cols;
  int step;                // 0: out = X;  1: out = keep * out - rate * X
  float keep, rate;
};

// Y = a X + P X;  LAST: into the result instead
template <class S, bool LAST>
__global__ __launch_bounds__(S::THREADS, 2) void apply_kernel(Mats q, int tm, int tn, float ca, Result res) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int im, in;
  tg::tile_of(blockIdx.x, tm, tn, im, in);
  const int b = blockIdx.y, m0 = im * S::BM, n0 = in * S::BN;
  const bf16_t* X = q.X + b * q.sx;
  f32x4 acc[S::MT][S::NT];
  tg::clear<S>(acc);
  tg::run<S, tg::KC, tg::KM>(tg::Operand{q.P + b * q.sg, q.ldg, q.m, 0}, tg::Operand{X, q.ldx, q.m, (int)q.ldx}, m0, n0, 0, (int)(q.ldg / 64), smem, acc);
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = (int)threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
  for (int x = 0; x < S::MT; ++x) {
    const int m = m0 + (wm * S::MT + x) * 16 + l16;
    if (m >= q.m) continue;
#pragma unroll
    for (int y = 0; y < S::NT; ++y) {
      const int n = n0 + (wn * S::NT + y) * 16 + 4 * l4;
      if (n >= q.ldx / 2) continue;
      float v[4];
      tg::load4<2>(X + m * q.ldx, n, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = n + e < q.n ? fmaf(ca, v[e], acc[x][y][e]) : 0.f;
      if constexpr (!LAST) {
        tg::store4<2>(q.Y + b * q.sx + m * q.ldx, n, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (n + e >= q.n) continue;
          const int64_t at = (int64_t)b * res.rows * res.cols + (res.tall ? (int64_t)(n + e) * res.cols + m : (int64_t)m * res.cols + n + e);
          if (res.out_bf16) {
            bf16_t* o = reinterpret_cast<bf16_t*>(res.out) + at;
            *o = f2bf(res.step ? fmaf(-res.rate, v[e], res.keep * bf2f(*o)) : v[e]);
          } else {
            float* o = reinterpret_cast<float*>(res.out) + at;
            *o = fmaf(-res.rate, v[e], res.keep * *o);
          }
        }
      }
    }
  }
}

typedef tg::Shape<256, 256, 2, 4, 2, 2> ShapeL;
typedef tg::Shape<128, 128, 2, 2, 2, 2> ShapeM;
typedef tg::Shape<64, 64, 2, 2, 2, 4> ShapeS;

template <typename K>
int allow_lds(K kernel, int bytes) {
  SGPO_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return SGPO_OK;
}
#define ALLOW(kernel, bytes)                                           \
  do {                                                                 \
    static bool done = false;                                          \
    if (!done) { const int rc_ = allow_lds(kernel, bytes); if (rc_) return rc_; done = true; } \
  } while (0)

template <class S, bool POLY>
int symmetric(const Mats& q, int batch, float cb, float cc, hipStream_t st) {
  const int t = (q.m + S::BM - 1) / S::BM;
  ALLOW((symmetric_kernel<S, POLY>), S::LDS);
  hipLaunchKernelGGL((symmetric_kernel<S, POLY>), dim3((unsigned)(t * (t + 1) / 2), batch), dim3(S::THREADS), S::LDS, st, q, t, cb, cc);
  return SGPO_OK;
}
template <class S, bool LAST>
int apply(const Mats& q, int batch, float ca, const Result& r, hipStream_t st) {
  const int tm = (q.m + S::BM - 1) / S::BM, tn = (q.n + S::BN - 1) / S::BN;
  ALLOW((apply_kernel<S, LAST>), S::LDS);
  hipLaunchKernelGGL((apply_kernel<S, LAST>), dim3((unsigned)tm * tn, batch), dim3(S::THREADS), S::LDS, st, q, tm, tn, ca, r);
  return SGPO_OK;
}

int pick_symmetric(int64_t m, int64_t batch) {
  auto tri = [&](int64_t s) { const int64_t t = (m + s - 1) / s; return batch * t * (t + 1) / 2; };
  return tri(256) >= 160 ? 2 : tri(128) >= 160 ? 1 : 0;
}
int pick_full(int64_t m, int64_t n, int64_t batch) {
  auto cnt = [&](int64_t s) { return batch * ((m + s - 1) / s) * ((n + s - 1) / s); };
  return cnt(256) >= 160 ? 2 : cnt(128) >= 160 ? 1 : 0;
}

struct Sizes { int m, n; int64_t ldx, ldg; size_t x, g, off_x, off_y, off_g, off_p, bytes; };
Sizes sizes(int batch, int rows, int cols) {
  Sizes s;
  s.m = rows < cols ? rows : cols;
  s.n = rows < cols ? cols : rows;
  s.ldx = round_up(s.n, 32) * 2;
  s.ldg = round_up(s.m, 32) * 2;
  s.x = (size_t)s.m * s.ldx; s.g = (size_t)s.m * s.ldg;
  size_t at = 0;
  auto take = [&](size_t n) { const size_t o = at; at += (n + 255) & ~(size_t)255; return o; };
  take((size_t)batch * PARTS * 8);
  s.off_x = take(batch * s.x * 2); s.off_y = take(batch * s.x * 2);
  s.off_g = take(batch * s.g * 2); s.off_p = take(batch * s.g * 2);
  s.bytes = at;
  return s;
}

template <typename T>
int orthogonalise(const Source& src, int batch, const float* coef, int steps, double eps, Result res, char* ws, hipStream_t st) {
  const Sizes z = sizes(batch, src.rows, src.cols);
  double* part = reinterpret_cast<double*>(ws);
  Mats q{(bf16_t*)(ws + z.off_x), (bf16_t*)(ws + z.off_y), (bf16_t*)(ws + z.off_g), (bf16_t*)(ws + z.off_p), z.ldx, z.ldg, (int64_t)z.x, (int64_t)z.g, z.m, z.n};
  res.tall = src.rows > src.cols; res.rows = src.rows; res.cols = src.cols;
  hipLaunchKernelGGL((square_kernel<T>), dim3(PARTS, batch), dim3(256), 0, st, src, part);
  const dim3 grid((unsigned)((z.ldx / 2 + 63) / 64), (unsigned)((z.m + 63) / 64), batch);
  if (res.tall) hipLaunchKernelGGL((load_kernel<T, true>), grid, dim3(256), 0, st, src, part, eps, q.X, z.m, z.n, z.ldx, (int64_t)z.x);
  else hipLaunchKernelGGL((load_kernel<T, false>), grid, dim3(256), 0, st, src, part, eps, q.X, z.m, z.n, z.ldx, (int64_t)z.x);
  const int cs = pick_symmetric(z.m, batch), cf = pick_full(z.m, z.n, batch);
  for (int k = 0; k < steps; ++k) {
    const float a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2];
    int rc = cs == 2 ? symmetric<ShapeL, false>(q, batch, b, c, st) : cs == 1 ? symmetric<ShapeM, false>(q, batch, b, c, st) : symmetric<ShapeS, false>(q, batch, b, c, st);
    if (rc) return rc;
    rc = cs == 2 ? symmetric<ShapeL, true>(q, batch, b, c, st) : cs == 1 ? symmetric<ShapeM, true>(q, batch, b, c, st) : symmetric<ShapeS, true>(q, batch, b, c, st);
    if (rc) return rc;
    if (k + 1 < steps) rc = cf == 2 ? apply<ShapeL, false>(q, batch, a, res, st) : cf == 1 ? apply<ShapeM, false>(q, batch, a, res, st) : apply<ShapeS, false>(q, batch, a, res, st);
    else rc = cf == 2 ? apply<ShapeL, true>(q, batch, a, res, st) : cf == 1 ? apply<ShapeM, true>(q, batch, a, res, st) : apply<ShapeS, true>(q, batch, a, res, st);
    if (rc) return rc;
    bf16_t* t = q.X; q.X = q.Y; q.Y = t;
  }
  SGPO_CHECK_HIP(hipGetLastError());
  return SGPO_OK;
}

int check_sizes(int batch, int rows, int cols, int steps, const float* coef) {
  SGPO_REQUIRE(batch >= 0 && rows >= 0 && cols >= 0, "newton_schulz: negative size");
  SGPO_REQUIRE(batch <= 65535 && rows <= (1 << 17) && cols <= (1 << 17), "newton_schulz: %d matrices of %d x %d over the supported range", batch, rows, cols);
  SGPO_REQUIRE(steps >= 1 && steps <= 64 && coef, "newton_schulz: 1 to 64 coefficient triples are needed, got %d", steps);
  return SGPO_OK;
}

}  // namespace

extern "C" size_t sgpo_newton_schulz_workspace_bytes(int batch, int rows, int cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  return sizes(batch, rows, cols).bytes;
}

extern "C" int sgpo_newton_schulz(const void* update, int dtype, int batch, int rows, int cols, int64_t stride_b, int64_t ld, const float* coefficients,
                                  int steps, float eps, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_sizes(batch, rows, cols, steps, coefficients);
  if (rc) return rc;
  SGPO_REQUIRE(dtype == SGPO_DTYPE_F32 || dtype == SGPO_DTYPE_BF16, "newton_schulz: unknown dtype %d", dtype);
  if (!batch || !rows || !cols) return SGPO_OK;
  SGPO_REQUIRE(update && out && workspace, "newton_schulz: null argument");
  SGPO_REQUIRE(ld >= cols || rows == 1, "newton_schulz: row pitch %lld below %d columns", (long long)ld, cols);
  const size_t need = sgpo_newton_schulz_workspace_bytes(batch, rows, cols);
  if (workspace_bytes < need) { sgpo_set_error("newton_schulz: workspace %zu < %zu", workspace_bytes, need); return SGPO_ERR_WORKSPACE; }
  const Source s{update, nullptr, 0.f, 0, stride_b, ld, rows, cols};
  const Result r{out, 1, 0, 0, 0, 0, 0.f, 0.f};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == SGPO_DTYPE_BF16 ? orthogonalise<bf16_t>(s, batch, coefficients, steps, eps, r, (char*)workspace, st)
                                  : orthogonalise<float>(s, batch, coefficients, steps, eps, r, (char*)workspace, st);
}

extern "C" int sgpo_muon_step(void* weight, int weight_dtype, const void* grad, int grad_dtype, float* momentum_buffer, int batch, int rows, int cols,
                              float lr, float momentum, int nesterov, float weight_decay, const float* coefficients, int steps, float eps, void* workspace,
                              size_t workspace_bytes, void* stream) {
  int rc = check_sizes(batch, rows, cols, steps, coefficients);
  if (rc) return rc;
  SGPO_REQUIRE((weight_dtype == SGPO_DTYPE_F32 || weight_dtype == SGPO_DTYPE_BF16) && (grad_dtype == SGPO_DTYPE_F32 || grad_dtype == SGPO_DTYPE_BF16),
               "muon_step: unknown dtype %d / %d", weight_dtype, grad_dtype);
  if (!batch || !rows || !cols) return SGPO_OK;
  SGPO_REQUIRE(weight && grad && momentum_buffer && workspace, "muon_step: null argument");
  const size_t need = sgpo_newton_schulz_workspace_bytes(batch, rows, cols);
  if (workspace_bytes < need) { sgpo_set_error("muon_step: workspace %zu < %zu", workspace_bytes, need); return SGPO_ERR_WORKSPACE; }
  const Source s{grad, momentum_buffer, momentum, nesterov != 0, (int64_t)rows * cols, cols, rows, cols};
  const double ratio = rows > cols ? (double)rows / cols : 1.0;
  const Result r{weight, weight_dtype == SGPO_DTYPE_BF16, 0, 0, 0, 1, (float)(1.0 - (double)lr * weight_decay), (float)(lr * sqrt(ratio))};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return grad_dtype == SGPO_DTYPE_BF16 ? orthogonalise<bf16_t>(s, batch, coefficients, steps, eps, r, (char*)workspace, st)
                                       : orthogonalise<float>(s, batch, coefficients, steps, eps, r, (char*)workspace, st);
}
