// Orthogonalised updates by Newton-Schulz products, and the optimiser step around them.
//
//   X_0 = U / (|U|_F + eps)
//   G = X X^T,  P = a I + b G + c G G,  X <- P X          once per coefficient triple (a, b, c)
//   (G = X^T X and X <- X P where X has more rows than columns: the products' operands are read by rows or by columns as stored, nothing is transposed)
// which moves every singular value of X towards 1 by the odd polynomial a s + b s^3 + c s^5 and leaves the singular vectors.
//   step:  buf <- mu buf + grad,  U = grad + mu buf (or buf),  W <- (1 - lr wd) W - lr sqrt(max(1, rows / cols)) X
//
// Bound by the matrix cores: per triple m^2 n + m^3 + 2 m^2 n operations, the two symmetric products at half (one triangle of tiles,
// each written twice).  X, G and P are held as two bf16 planes, about 17 bits (tile_gemm.h; fp32 on the second way below): in one plane the rounding of X
// pollutes the directions of small singular values, which the polynomial then multiplies by up to a^5 = 485 (relative error of
// the result 2e-2 on Gaussian updates, against 3e-5 with two planes; the result is rounded to bf16, 2e-3).
// The squared norm is summed in 64 bits: it neither overflows nor depends on how the update is cut.  An infinity or NaN in an update
// makes its whole result NaN.
// Three ways: both sides small, one workgroup and launch per matrix; one side small, iteration on d x d matrices; tiles over the device.
#include "../../include/sgpo_hip.h"
#include "tile_gemm.h"

namespace {

constexpr int PARTS = 512;   // partial sums of a matrix's squared norm: at most, and a multiple of 64

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
  int rows, cols, flat;    // flat: a matrix of grad is contiguous
};

template <typename T>
__device__ __forceinline__ float update_at(const Source& s, int b, int r, int c) {   // after the buffer's own update
  const float g = up<T>(reinterpret_cast<const T*>(s.grad)[b * s.stride_b + r * s.ld + c]);
  if (!s.buf) return g;
  const float m = s.buf[((int64_t)b * s.rows + r) * s.cols + c];
  return s.nesterov ? fmaf(s.momentum, m, g) : m;
}

// four consecutive elements of a gradient's row, of any alignment
__device__ __forceinline__ void grad4(const float* p, float (&g)[4]) { __builtin_memcpy(g, p, 16); }
__device__ __forceinline__ void grad4(const bf16_t* p, float (&g)[4]) {
  uint32_t v[2];
  __builtin_memcpy(v, p, 8);
  g[0] = bf2f(v[0] & 0xffff); g[1] = bf2f(v[0] >> 16); g[2] = bf2f(v[1] & 0xffff); g[3] = bf2f(v[1] >> 16);
}
// elements (r, c .. c + 3) of the update, those that exist; after the buffer's own update
template <typename T>
__device__ __forceinline__ void update4(const Source& s, int b, int r, int c, float (&v)[4]) {
  if (c + 4 <= s.cols) {
    grad4(reinterpret_cast<const T*>(s.grad) + b * s.stride_b + r * s.ld + c, v);
    if (s.buf) {
      f32x4 m;
      __builtin_memcpy(&m, s.buf + ((int64_t)b * s.rows + r) * s.cols + c, 16);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = s.nesterov ? fmaf(s.momentum, m[q], v[q]) : m[q];
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = c + q < s.cols ? update_at<T>(s, b, r, c + q) : 0.f;
  }
}

// momentum buffer, and partial sums of the update's squares; four elements at a time where a matrix is contiguous
template <typename T>
__global__ __launch_bounds__(256) void square_kernel(Source s, double* part) {
  const int b = blockIdx.y;
  const uint32_t total = (uint32_t)s.rows * (uint32_t)s.cols;
  const T* grad = reinterpret_cast<const T*>(s.grad) + b * s.stride_b;
  float* buf = s.buf ? s.buf + (int64_t)b * total : nullptr;
  double sum = 0.0;
  uint32_t done = 0;
  if (s.flat) {
    done = total / 4 * 4;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < total / 4; i += gridDim.x * 256) {
      float g[4];
      grad4(grad + (size_t)i * 4, g);
      if (buf) {
        f32x4 m;
        __builtin_memcpy(&m, buf + (size_t)i * 4, 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          m[q] = fmaf(s.momentum, m[q], g[q]);
          g[q] = s.nesterov ? fmaf(s.momentum, m[q], g[q]) : m[q];
        }
        __builtin_memcpy(buf + (size_t)i * 4, &m, 16);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) sum += (double)g[q] * g[q];
    }
  }
  for (uint32_t i = done + blockIdx.x * 256 + threadIdx.x; i < total; i += gridDim.x * 256) {
    const uint32_t r = i / (uint32_t)s.cols, c = i - r * (uint32_t)s.cols;
    if (buf) buf[i] = fmaf(s.momentum, buf[i], up<T>(grad[r * s.ld + c]));
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

__device__ __forceinline__ float inverse_norm(const double* part, int parts, double eps) {   // every lane of the wave calls it
  double s = 0.0;
  for (int i = threadIdx.x & 63; i < parts; i += 64) s += part[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  return (float)(1.0 / (sqrt(s) + eps));
}

// X planes of the scaled update, zero in the padding columns
template <typename T>
__global__ __launch_bounds__(256) void load_kernel(Source s, const double* part, int parts, double eps, bf16_t* X, int64_t ldx, int64_t bstride) {
  const int b = blockIdx.y;
  const float inv = inverse_norm(part + b * PARTS, parts, eps);
  const uint32_t quads = (uint32_t)(ldx / 8), total = (uint32_t)s.rows * quads;
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < total; i += gridDim.x * 256) {
    const int r = (int)(i / quads), c = (int)(i - (uint32_t)r * quads) * 4;
    float v[4];
    update4<T>(s, b, r, c, v);
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] *= inv;
    tg::store4<2, true>(X + b * bstride + r * ldx, c, v);
  }
}

struct Mats {
  bf16_t *X, *Y, *G, *P;      // planes: X, Y [rows][cols], G, P [d][d], d the shorter side
  int64_t ldx, ldg, sx, sg;   // row pitch and batch stride, stored elements
  int rows, cols, d;
};

// Workgroup -> (matrix, tile): workgroups with equal id % 8 share an XCD and its L2, and each XCD takes one contiguous run of the list of all
// matrices' tiles, so that a matrix is read into few L2s (512 x 2048, eight of them: each XCD its own matrix).
__device__ __forceinline__ void contiguous(int id, int total, int per, int& b, int& t) {
  const int q = total >> 3, r = total & 7, x = id & 7;
  t = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (id >> 3);
  b = t / per;
  t -= b * per;
}
// tile (i, j), i <= j, of the triangle, row by row
__device__ __forceinline__ void triangle(int t, int tiles, int& i, int& j) {
  i = 0;
  while (t >= tiles - i) { t -= tiles - i; ++i; }
  j = i + t;
}

// K cut over gridDim.y: fp32 sums [cut][matrix][d][pitch], in the tiles of the triangle
struct Slabs {
  float* out;        // null: not cut
  int steps, pitch;  // K steps per cut
};

enum { WIDE = 0, TALL = 1, POLY = 2 };   // G = X X^T;  G = X^T X;  P = a I + b G + c G G

// One triangle of tiles, each also written transposed (element by element: taking the transposed tile through LDS and out in whole lines
// measured the same, 60 us either way for 512 x 1536 in 192 x 192 tiles)
template <class S, int MODE>
__global__ __launch_bounds__(S::WG_THREADS, 2) void symmetric_kernel(Mats q, int tiles, float ca, float cb, float cc, Slabs slabs) {
  static_assert(S::BM == S::BN && S::PL == 2, "square tiles of two planes");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int i, j, b, t;
  contiguous(blockIdx.x, gridDim.x, tiles * (tiles + 1) / 2, b, t);
  triangle(t, tiles, i, j);
  const int m0 = i * S::BM, n0 = j * S::BN;
  const bf16_t* G = q.G + b * q.sg;
  f32x4 acc[S::MT][S::NT];
  tg::clear<S>(acc);
  if constexpr (MODE == TALL) {
    const tg::Operand o{q.X + b * q.sx, q.ldx, q.rows, (int)q.ldx};
    const int nk = (q.rows + 31) / 32, k0 = slabs.out ? blockIdx.y * slabs.steps : 0;
    tg::run<S, tg::KM, tg::KM>(o, o, m0, n0, k0, slabs.out ? min(slabs.steps, nk - k0) : nk, smem, acc);
  } else {
    const tg::Operand o{MODE == POLY ? G : q.X + b * q.sx, MODE == POLY ? q.ldg : q.ldx, q.d, 0};
    const int nk = (int)(o.ld / 64), k0 = MODE != POLY && slabs.out ? blockIdx.y * slabs.steps : 0;
    tg::run<S, tg::KC, tg::KC>(o, o, m0, n0, k0, MODE != POLY && slabs.out ? min(slabs.steps, nk - k0) : nk, smem, acc);
  }
  bf16_t* dst = (MODE == POLY ? q.P : q.G) + b * q.sg;
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4, wm = S::wave() / S::WN, wn = S::wave() % S::WN;
#pragma unroll
  for (int x = 0; x < S::MT; ++x) {
    const int m = m0 + (wm * S::MT + x) * 16 + l16;
#pragma unroll
    for (int y = 0; y < S::NT; ++y) {
      if (!S::owns(x, y)) continue;
      const int n = n0 + (wn * S::NT + y) * 16 + 4 * l4;
      if (MODE != POLY && slabs.out) {
        if (m < q.d && n < slabs.pitch) *reinterpret_cast<f32x4*>(slabs.out + (((int64_t)blockIdx.y * (gridDim.x / (tiles * (tiles + 1) / 2)) + b) * q.d + m) * slabs.pitch + n) = acc[x][y];
        continue;
      }
      float v[4] = {acc[x][y][0], acc[x][y][1], acc[x][y][2], acc[x][y][3]};
      if (m < q.d && n < q.ldg / 2) {
        if constexpr (MODE == POLY) {
          float g[4];
          tg::load4<2>(G + m * q.ldg, n, g);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = fmaf(cb, g[e], cc * v[e]) + (m == n + e ? ca : 0.f);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) if (n + e >= q.d) v[e] = 0.f;
        tg::store4<2, true>(dst + m * q.ldg, n, v);
      }
      if (i != j && m < q.ldg / 2) {   // the mirror image: row n + e, column m
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < q.d) {
            float pl[2];
            tg::split<2, true>(m < q.d ? v[e] : 0.f, pl);
            bf16_t* at = dst + (n + e) * q.ldg + (m >> 5) * 64 + (m & 31);
            at[0] = f2bf(pl[0]);
            at[32] = f2bf(pl[1]);
          }
      }
    }
  }
}

// G from the cuts' sums; side: of the triangle's tiles
__global__ __launch_bounds__(256) void join_kernel(Mats q, Slabs slabs, int cuts, int side) {
  const int b = blockIdx.y, quads = (int)(q.ldg / 8);
  const int64_t stride = (int64_t)gridDim.y * q.d * slabs.pitch;
  const float* src = slabs.out + (int64_t)b * q.d * slabs.pitch;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < q.d * quads; i += gridDim.x * 256) {
    const int r = i / quads, c = (i - r * quads) * 4;
    if (c / side < r / side) continue;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (c < slabs.pitch) {
      const float* at = src + (int64_t)r * slabs.pitch + c;
#pragma unroll 8
      for (int k = 0; k < cuts; ++k) v += *reinterpret_cast<const f32x4*>(at + k * stride);
    }
    const float w[4] = {c < q.d ? v[0] : 0.f, c + 1 < q.d ? v[1] : 0.f, c + 2 < q.d ? v[2] : 0.f, c + 3 < q.d ? v[3] : 0.f};
    bf16_t* g = q.G + b * q.sg;
    tg::store4<2, true>(g + r * q.ldg, c, w);
    if (c / side > r / side) {   // the tile below the diagonal: 2-byte stores, where reading the sums transposed took 13 us (100 x 100, 32 cuts)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c + e >= q.d) break;
        float pl[2];
        tg::split<2, true>(w[e], pl);
        bf16_t* to = g + (c + e) * q.ldg + (r >> 5) * 64 + (r & 31);
        to[0] = f2bf(pl[0]);
        to[32] = f2bf(pl[1]);
      }
    }
  }
}

struct Result {
  void* out;               // bf16 [batch][rows][cols], or the weight
  int out_bf16;
  int rows, cols;
  int step;                // 0: out = X;  1: out = keep * out - rate * X
  float keep, rate;
};

__device__ __forceinline__ float result(const Result& r, float old, float v) { return r.step ? fmaf(-r.rate, v, r.keep * old) : v; }
// elements (m, n .. n + 3) of X, those that exist
__device__ __forceinline__ void store_result(const Result& r, int b, int m, int n, const float (&v)[4]) {
  const int64_t at = ((int64_t)b * r.rows + m) * r.cols + n;
  if (r.out_bf16) {
    bf16_t* o = reinterpret_cast<bf16_t*>(r.out) + at;
    if (n + 4 <= r.cols) {
      uint32_t w[2] = {0, 0};
      if (r.step) __builtin_memcpy(w, o, 8);
      w[0] = pack_bf16x2(result(r, bf2f(w[0] & 0xffff), v[0]), result(r, bf2f(w[0] >> 16), v[1]));
      w[1] = pack_bf16x2(result(r, bf2f(w[1] & 0xffff), v[2]), result(r, bf2f(w[1] >> 16), v[3]));
      __builtin_memcpy(o, w, 8);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) if (n + e < r.cols) o[e] = f2bf(result(r, r.step ? bf2f(o[e]) : 0.f, v[e]));
    }
  } else {   // only a step writes fp32
    float* o = reinterpret_cast<float*>(r.out) + at;
    if (n + 4 <= r.cols) {
      f32x4 w;
      __builtin_memcpy(&w, o, 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = result(r, w[e], v[e]);
      __builtin_memcpy(o, &w, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) if (n + e < r.cols) o[e] = result(r, o[e], v[e]);
    }
  }
}

// Matrices of at most 128 x 128: everything in one launch, one workgroup per matrix.  X stays in registers in fp32 (the layout of the products'
// results); its planes, and those of G and then P, pass through LDS.  One LDS image serves both as rows (X X^T, G G, P .) and, by
// transposed reads, as columns (. X): rows of 2 * E planes elements, their 16-B chunks permuted by a function of the row that
// keeps both kinds of read off each other's banks.  Bound by the chain of 3 dependent products per triple, each a few LDS round trips.
template <int E>
struct Small {
  static constexpr int WAVES_M = 4, WAVES_N = 4, THREADS = 64 * WAVES_M * WAVES_N;
  static constexpr int MT = E / WAVES_M / 16, NT = E / WAVES_N / 16;
  static constexpr int ROWB = E * 4, IMAGE = E * ROWB, IMAGES = 4 * IMAGE <= 163840 ? 4 : 2, LDS = IMAGES * IMAGE;
  typedef f32x4 Acc[MT][NT];
  __device__ static __forceinline__ int swz(int row) { return ((row & 1) << 1) | ((row & 2) << 1) | ((row & 8)) | ((row >> 2) & 1); }
  // byte of element (row, e) of plane 0; its 16-B chunk holds e .. e + 7 of one plane, plane 1 is 4 chunks on
  __device__ static __forceinline__ int at(int row, int e, int plane) { return row * ROWB + ((((e >> 5) * 8 + plane * 4 + ((e >> 3) & 3)) ^ swz(row)) << 4) + (e & 7) * 2; }
  __device__ static __forceinline__ bf16x8 row_fragment(const char* img, int row, int slice, int plane, int l4) {
    return *reinterpret_cast<const bf16x8*>(img + at(row, slice * 32 + l4 * 8, plane));
  }
  __device__ static __forceinline__ bf16x8 col_fragment(const char* img, int col16, int slice, int plane, int l16, int l4) {
    const int row = slice * 32 + l4 * 8 + (l16 >> 2), e = col16 * 16 + (l16 & 3) * 4;
    const tg::s16x4 lo = tg::read_tr((tg::lds_tr_t)(img + at(row, e, plane)));
    const tg::s16x4 hi = tg::read_tr((tg::lds_tr_t)(img + at(row + 4, e, plane)));
    const tg::s16x8 v = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    return *reinterpret_cast<const bf16x8*>(&v);
  }
  // r = A B^T (COLS false: both images by rows) or A B (B by columns), k < 32 * slices
  template <bool COLS>
  __device__ static __forceinline__ void product(const char* A, const char* B, int slices, Acc& r, int wm, int wn, int l16, int l4) {
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
      for (int y = 0; y < NT; ++y) r[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < E / 32; ++s) {   // unrolled: the fragments' addresses are then formed once for all triples
      if (s >= slices) break;
      bf16x8 a[2][MT], b[2][NT];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int x = 0; x < MT; ++x) a[p][x] = row_fragment(A, (wm * MT + x) * 16 + l16, s, p, l4);
#pragma unroll
        for (int y = 0; y < NT; ++y) b[p][y] = COLS ? col_fragment(B, wn * NT + y, s, p, l16, l4) : row_fragment(B, (wn * NT + y) * 16 + l16, s, p, l4);
      }
#pragma unroll
      for (int k = 2; k >= 0; --k)   // the two mixed pairs, then the high one
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
          for (int y = 0; y < NT; ++y) r[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[k == 1][y], a[k == 2][x], r[x][y], 0, 0, 0);
    }
  }
  __device__ static __forceinline__ void put(char* img, const Acc& v, int wm, int wn, int l16, int l4) {
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
      for (int y = 0; y < NT; ++y) {
        const int row = (wm * MT + x) * 16 + l16, e = (wn * NT + y) * 16 + 4 * l4;
        float pl[4][2];
#pragma unroll
        for (int q = 0; q < 4; ++q) tg::split<2, true>(v[x][y][q], pl[q]);
#pragma unroll
        for (int p = 0; p < 2; ++p)
          *reinterpret_cast<uint2*>(img + at(row, e, p)) = make_uint2(pack_bf16x2(pl[0][p], pl[1][p]), pack_bf16x2(pl[2][p], pl[3][p]));
      }
  }
};

struct Table { float v[3 * 64]; };

template <typename T, int E>
__global__ __launch_bounds__(Small<E>::THREADS, 1) void small_kernel(Source s, int m, int n, int tall, Table coef, int steps, double eps, Result res) {
  typedef Small<E> K;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ double share[K::THREADS / 64];
  const int b = blockIdx.x, lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wm = wave / K::WAVES_N, wn = wave % K::WAVES_N;
  typename K::Acc x, g, h;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < K::MT; ++i)
#pragma unroll
    for (int j = 0; j < K::NT; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int mm = (wm * K::MT + i) * 16 + l16, nn = (wn * K::NT + j) * 16 + 4 * l4 + q;
        float u = 0.f;
        if (mm < m && nn < n) {
          const int r = tall ? nn : mm, c = tall ? mm : nn;
          if (s.buf) {
            float* at = s.buf + ((int64_t)b * s.rows + r) * s.cols + c;
            *at = fmaf(s.momentum, *at, up<T>(reinterpret_cast<const T*>(s.grad)[b * s.stride_b + r * s.ld + c]));
          }
          u = update_at<T>(s, b, r, c);
        }
        x[i][j][q] = u;
        sum += (double)u * u;
      }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) share[wave] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int w = 0; w < K::THREADS / 64; ++w) sum += share[w];
  const float inv = (float)(1.0 / (sqrt(sum) + eps));
#pragma unroll
  for (int i = 0; i < K::MT; ++i)
#pragma unroll
    for (int j = 0; j < K::NT; ++j) x[i][j] *= inv;
  const int sm = (m + 31) >> 5, sn = (n + 31) >> 5;   // k slices
  // Four images (X and the next X, G, P) need one barrier per product; where only two fit, what overwrites an image waits for its readers.
  constexpr bool ROOM = K::IMAGES == 4;
  char *X = smem, *G = smem + K::IMAGE, *P = ROOM ? smem + 2 * K::IMAGE : G, *next = ROOM ? smem + 3 * K::IMAGE : X;
  K::put(X, x, wm, wn, l16, l4);
  __syncthreads();
  for (int k = 0; k < steps; ++k) {
    const float ca = coef.v[3 * k], cb = coef.v[3 * k + 1], cc = coef.v[3 * k + 2];
    K::template product<false>(X, X, sn, g, wm, wn, l16, l4);
    K::put(G, g, wm, wn, l16, l4);
    __syncthreads();
    K::template product<false>(G, G, sm, h, wm, wn, l16, l4);
#pragma unroll
    for (int i = 0; i < K::MT; ++i)
#pragma unroll
      for (int j = 0; j < K::NT; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) h[i][j][q] = fmaf(cb, g[i][j][q], cc * h[i][j][q]);
    if (!ROOM) __syncthreads();
    K::put(P, h, wm, wn, l16, l4);
    __syncthreads();
    K::template product<true>(P, X, sm, g, wm, wn, l16, l4);
#pragma unroll
    for (int i = 0; i < K::MT; ++i)
#pragma unroll
      for (int j = 0; j < K::NT; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) x[i][j][q] = fmaf(ca, x[i][j][q], g[i][j][q]);
    if (k + 1 == steps) break;
    if (!ROOM) __syncthreads();
    K::put(next, x, wm, wn, l16, l4);
    __syncthreads();
    char* t = X; X = next; next = t;
  }
#pragma unroll
  for (int i = 0; i < K::MT; ++i)
#pragma unroll
    for (int j = 0; j < K::NT; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int mm = (wm * K::MT + i) * 16 + l16, nn = (wn * K::NT + j) * 16 + 4 * l4 + q;
        if (mm >= m || nn >= n) continue;
        const int64_t at = ((int64_t)b * s.rows + (tall ? nn : mm)) * s.cols + (tall ? mm : nn);
        if (res.out_bf16) {
          bf16_t* o = reinterpret_cast<bf16_t*>(res.out) + at;
          *o = f2bf(result(res, res.step ? bf2f(*o) : 0.f, x[i][j][q]));
        } else {
          float* o = reinterpret_cast<float*>(res.out) + at;
          *o = result(res, *o, x[i][j][q]);
        }
      }
}

// Y = P X, or X P if TALLX;  LAST: into the result instead
template <class S, bool TALLX, bool LAST>
__global__ __launch_bounds__(S::WG_THREADS, 2) void apply_kernel(Mats q, int tm, int tn, Result res) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int b, t;
  contiguous(blockIdx.x, gridDim.x, tm * tn, b, t);
  const int band = 8 * tn, first = t / band * 8, h = min(8, tm - first);   // bands of 8 row tiles
  const int im = first + t % band % h, in = t % band / h;
  const int m0 = im * S::BM, n0 = in * S::BN;
  const bf16_t *X = q.X + b * q.sx, *P = q.P + b * q.sg;
  f32x4 acc[S::MT][S::NT];
  tg::clear<S>(acc);
  if constexpr (TALLX) tg::run<S, tg::KC, tg::KC, !LAST>(tg::Operand{X, q.ldx, q.rows, 0}, tg::Operand{P, q.ldg, q.d, 0}, m0, n0, 0, (int)(q.ldg / 64), smem, acc);   // P is symmetric
  else tg::run<S, tg::KC, tg::KM, !LAST>(tg::Operand{P, q.ldg, q.d, 0}, tg::Operand{X, q.ldx, q.d, (int)q.ldx}, m0, n0, 0, (int)(q.ldg / 64), smem, acc);
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4, wm = S::wave() / S::WN, wn = S::wave() % S::WN;
  const int pad = (int)(q.ldx / 2);
#pragma unroll
  for (int x = 0; x < S::MT; ++x) {
    const int m = m0 + (wm * S::MT + x) * 16 + l16;
    const bool row = m < q.rows;
    float w[S::NT][4];
#pragma unroll
    for (int y = 0; y < S::NT; ++y) {
      if (!S::template owns<!LAST>(x, y)) continue;
      const int n = n0 + (wn * S::NT + y) * 16 + 4 * l4;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[y][e] = n + e < q.cols ? acc[x][y][e] : 0.f;
      if (LAST && row && n < q.cols) store_result(res, b, m, n, w[y]);
    }
    if constexpr (!LAST) {
      bf16_t* at = q.Y + b * q.sx + m * q.ldx;
#pragma unroll
      for (int y = 0; y < S::NT; y += 2) {
        if (!S::template owns<!LAST>(x, y)) continue;
        const int e = n0 + (wn * S::NT + y) * 16;
        if (y + 1 < S::NT && e % 32 == 0) tg::store_pair<2, true>(at, e, w[y], w[y + 1 < S::NT ? y + 1 : y], l4, row && e < pad);
        else {
          if (row && e < pad) tg::store4<2, true>(at, e + 4 * l4, w[y]);
          if (y + 1 < S::NT && row && e + 16 < pad) tg::store4<2, true>(at, e + 16 + 4 * l4, w[y + 1 < S::NT ? y + 1 : y]);
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ long and narrow updates
// At most 64 rows (or columns) and more of the other: the iteration runs on d x d matrices.  X_k = Q_k X_0 with Q a polynomial in G_0 = X_0 X_0^T, so that
//   P = a I + b G + c G G,   Q <- P Q,   G <- P G P
// needs nothing of length n: X_0 is read for G_0 and again for the result Q X_0.  G's rounding grows by a^2 per triple in the directions of small
// singular values (where P's is read off it), so G is formed afresh from Q X_0 before that reaches GROWTH; five triples of the default: after three.
// Everything in fp32 on the fp32 matrix instructions (before the last rounding the result's relative error is 1e-6 on Gaussian updates and 1e-4 on nearly
// rank-one ones, the same with G formed afresh at every triple; formed once, 1e-6 and 1e-3).  Six launches instead of 17 to 22.  Bound by the chain of
// products in one workgroup, 0.9 us each at 64 x 64 and half of it the matrix instructions, and by the launches (64 x 4096: two times 11 us of 52).
constexpr int NARROW = 64, NARROW_CHUNK = 64, NARROW_PITCH = NARROW_CHUNK + 4;
constexpr double GROWTH = 200.;
struct NarrowArgs {
  Source src;
  const double* part;    // of the squared norm
  int parts;
  double eps;
  int d, n, tall;        // shorter and longer side
  float* Q;              // [batch][D][D]
  float* sums;           // [batch][cuts][D][D]
  int chunks, per, cuts;
};

// a chunk of 64 of the n columns of X_0: four elements along a row of the update at a time, zero beyond it; 256 threads
template <int D> struct Chunk { float v[D * NARROW_CHUNK / 4 / 256][4]; };
template <int D>
__device__ __forceinline__ void narrow_place(bool tall, int k, int& i, int& j) {   // the k-th quad's first element: short index, and long one within the chunk
  const int e = k * 256 + threadIdx.x;
  i = tall ? e % (D / 4) * 4 : e / (NARROW_CHUNK / 4);
  j = tall ? e / (D / 4) : e % (NARROW_CHUNK / 4) * 4;
}
template <typename T, int D>
__device__ __forceinline__ void narrow_load(const NarrowArgs& p, int b, int chunk, Chunk<D>& to) {
  const Source& s = p.src;
  const int j0 = chunk * NARROW_CHUNK;
#pragma unroll
  for (int k = 0; k < D * NARROW_CHUNK / 4 / 256; ++k) {
    int i, j;
    narrow_place<D>(p.tall, k, i, j);
    const int r = p.tall ? j0 + j : i, c = p.tall ? i : j0 + j;
    float (&v)[4] = to.v[k];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = 0.f;
    if (r < s.rows) update4<T>(s, b, r, c, v);
  }
}
// into tile [D][NARROW_PITCH]: short index, long index
template <int D>
__device__ __forceinline__ void narrow_put(const NarrowArgs& p, const Chunk<D>& from, float inv, float* tile) {
#pragma unroll
  for (int k = 0; k < D * NARROW_CHUNK / 4 / 256; ++k) {
    int i, j;
    narrow_place<D>(p.tall, k, i, j);
    const float (&v)[4] = from.v[k];
    if (p.tall) {
#pragma unroll
      for (int q = 0; q < 4; ++q) tile[(i + q) * NARROW_PITCH + j] = v[q] * inv;
    } else {
      *reinterpret_cast<f32x4*>(tile + i * NARROW_PITCH + j) = f32x4{v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
    }
  }
}
// K elements of a row as a fragment: lane (l16, l4) holds k = l4 * K / 4 .., the same for both operands
template <int K>
__device__ __forceinline__ void narrow_row(const float* row, int l4, float (&f)[K / 4]) {
#pragma unroll
  for (int q = 0; q < K / 16; ++q) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(row + l4 * (K / 4) + 4 * q);
    f[4 * q] = v[0]; f[4 * q + 1] = v[1]; f[4 * q + 2] = v[2]; f[4 * q + 3] = v[3];
  }
}
// tile <- Q tile in place; wave w takes columns 16 w ..
template <int D>
__device__ __forceinline__ void narrow_turn(const float* Q, float* tile) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4, j = ((int)threadIdx.x >> 6) * 16 + l16;
  float f[D / 4];
#pragma unroll
  for (int k = 0; k < D / 4; ++k) f[k] = tile[(l4 * (D / 4) + k) * NARROW_PITCH + j];
  f32x4 acc[D / 16];
#pragma unroll
  for (int x = 0; x < D / 16; ++x) {
    float a[D / 4];
    narrow_row<D>(Q + (x * 16 + l16) * (D + 4), l4, a);
    acc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < D / 4; ++k) acc[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k], f[k], acc[x], 0, 0, 0);
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < D / 16; ++x)
#pragma unroll
    for (int q = 0; q < 4; ++q) tile[(x * 16 + 4 * l4 + q) * NARROW_PITCH + j] = acc[x][q];
  __syncthreads();
}
template <int D>
__device__ __forceinline__ void narrow_fetch(const float* from, float* Q) {
  for (int e = threadIdx.x; e < D * D / 4; e += 256)
    *reinterpret_cast<f32x4*>(Q + e / (D / 4) * (D + 4) + e % (D / 4) * 4) = *reinterpret_cast<const f32x4*>(from + e * 4);
}

// sums[b][cut] = X X^T over the cut's chunks, X = X_0 or Q X_0: the tiles on and over the diagonal
template <typename T, int D, bool TURN>
__global__ __launch_bounds__(256) void narrow_gram_kernel(NarrowArgs p) {
  __shared__ __attribute__((aligned(16))) float tile[D * NARROW_PITCH];
  __shared__ __attribute__((aligned(16))) float Q[TURN ? D * (D + 4) : 4];
  constexpr int TILES = D / 16 * (D / 16 + 1) / 2, MINE = (TILES + 3) / 4;   // 16 x 16 tiles of the triangle, and of a wave
  const int b = blockIdx.y, lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const float inv = inverse_norm(p.part + b * PARTS, p.parts, p.eps);
  if constexpr (TURN) narrow_fetch<D>(p.Q + (int64_t)b * D * D, Q);
  f32x4 acc[MINE];
#pragma unroll
  for (int t = 0; t < MINE; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int first = blockIdx.x * p.per, last = min(first + p.per, p.chunks);
  int x[MINE], y[MINE];
#pragma unroll
  for (int t = 0; t < MINE; ++t) triangle(min(wave + 4 * t, TILES - 1), D / 16, x[t], y[t]);
  Chunk<D> next;
  narrow_load<T, D>(p, b, first, next);
  for (int c = first; c < last; ++c) {
    __syncthreads();
    narrow_put<D>(p, next, inv, tile);
    __syncthreads();
    if (c + 1 < last) narrow_load<T, D>(p, b, c + 1, next);   // on its way while this one is multiplied
    if constexpr (TURN) narrow_turn<D>(Q, tile);
#pragma unroll
    for (int t = 0; t < MINE; ++t) {
      if (wave + 4 * t >= TILES) break;
      float a[NARROW_CHUNK / 4], f[NARROW_CHUNK / 4];
      narrow_row<NARROW_CHUNK>(tile + (x[t] * 16 + l16) * NARROW_PITCH, l4, a);
      narrow_row<NARROW_CHUNK>(tile + (y[t] * 16 + l16) * NARROW_PITCH, l4, f);
#pragma unroll
      for (int k = 0; k < NARROW_CHUNK / 4; ++k) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k], f[k], acc[t], 0, 0, 0);
    }
  }
  float* out = p.sums + ((int64_t)b * p.cuts + blockIdx.x) * D * D;
#pragma unroll
  for (int t = 0; t < MINE; ++t) {
    if (wave + 4 * t >= TILES) break;
#pragma unroll
    for (int q = 0; q < 4; ++q) out[(x[t] * 16 + 4 * l4 + q) * D + y[t] * 16 + l16] = acc[t][q];
  }
}

// the triples [k0, k1): Q <- P Q, G <- P G P; one workgroup per matrix, one wave per 16 x 16 tile of the triangle (64 x 64: the ten of them take the matrix
// instructions of three on a SIMD, all sixteen those of four).  The images hold whole matrices.  G, P and P G are symmetric but for rounding, which the mirrored
// triangle may decide; Q is not: P and Q of separate phases do not commute within what Q's large entries make of their rounding (on updates of low rank a
// mirrored Q was off by 7e-4 to 2e-2, against 3e-5), so Q is multiplied whole, in order, and kept transposed for its columns to be read as rows.
template <int D> constexpr int POLY_THREADS = D / 16 * (D / 16 + 1) / 2 * 64;
template <int D>
__global__ __launch_bounds__(POLY_THREADS<D>) void narrow_poly_kernel(NarrowArgs p, Table coef, int k0, int k1) {
  constexpr int PITCH = D + 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float *G = reinterpret_cast<float*>(smem), *P = G + D * PITCH, *M = P + D * PITCH, *Q = M + D * PITCH;
  const int b = blockIdx.x, lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  int x, y;
  triangle(__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), D / 16, x, y);
  const int row = x * 16 + 4 * l4, col = y * 16 + l16;
  const int row2 = y * 16 + 4 * l4, col2 = x * 16 + l16;   // the same lane's four elements of the tile's mirror image
  auto product = [&](const float* A, int i, const float* B, int j) {   // tile (i, j) of A B^T
    float a[D / 4], f[D / 4];
    narrow_row<D>(A + (i * 16 + l16) * PITCH, l4, a);
    narrow_row<D>(B + (j * 16 + l16) * PITCH, l4, f);
    f32x4 even = {0.f, 0.f, 0.f, 0.f}, odd = even;   // two chains
#pragma unroll
    for (int k = 0; k < D / 4; k += 2) {
      even = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k], f[k], even, 0, 0, 0);
      odd = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k + 1], f[k + 1], odd, 0, 0, 0);
    }
    return even + odd;
  };
  auto put = [&](float* img, const f32x4& v) {   // a symmetric matrix, both triangles
    *reinterpret_cast<f32x4*>(img + col * PITCH + row) = v;
    if (x == y) return;   // the tile itself is its mirror image
#pragma unroll
    for (int e = 0; e < 4; ++e) img[(row + e) * PITCH + col] = v[e];
  };
  f32x4 g = {0.f, 0.f, 0.f, 0.f}, q = g, q2 = g;   // q2: Q's tile (y, x)
  const float* from = p.sums + (int64_t)b * p.cuts * D * D + row * D + col;
#pragma unroll 4
  for (int c = 0; c < p.cuts; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) g[e] += from[(int64_t)c * D * D + e * D];
  put(G, g);
  auto put_q = [&]() {   // transposed
    *reinterpret_cast<f32x4*>(Q + col * PITCH + row) = q;
    if (x != y) *reinterpret_cast<f32x4*>(Q + col2 * PITCH + row2) = q2;
  };
  float* out = p.Q + (int64_t)b * D * D;
  if (k0 > 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { q[e] = out[(row + e) * D + col]; q2[e] = out[(row2 + e) * D + col2]; }
    put_q();
  }
  __syncthreads();
  for (int k = k0; k < k1; ++k) {
    const float ca = coef.v[3 * k], cb = coef.v[3 * k + 1], cc = coef.v[3 * k + 2];
    f32x4 h = product(G, x, G, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = fmaf(cb, g[e], cc * h[e]) + (row + e == col ? ca : 0.f);
    put(P, h);
    __syncthreads();
    if (k > 0) {
      q = product(P, x, Q, y);
      if (x != y) q2 = product(P, y, Q, x);
    } else {
      q = h;
      q2 = *reinterpret_cast<const f32x4*>(P + col2 * PITCH + row2);
    }
    if (k + 1 == k1) break;
    put(M, product(P, x, G, y));
    __syncthreads();
    g = product(P, x, M, y);
    put_q();
    put(G, g);
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) out[(row + e) * D + col] = q[e];
  if (x == y) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[(row2 + e) * D + col2] = q2[e];
}

// the result: Q X_0
template <typename T, int D>
__global__ __launch_bounds__(256) void narrow_apply_kernel(NarrowArgs p, Result res) {
  __shared__ __attribute__((aligned(16))) float tile[D * NARROW_PITCH];
  __shared__ __attribute__((aligned(16))) float Q[D * (D + 4)];
  const int b = blockIdx.y, chunk = blockIdx.x, j0 = chunk * NARROW_CHUNK;
  const float inv = inverse_norm(p.part + b * PARTS, p.parts, p.eps);
  narrow_fetch<D>(p.Q + (int64_t)b * D * D, Q);
  Chunk<D> here;
  narrow_load<T, D>(p, b, chunk, here);
  narrow_put<D>(p, here, inv, tile);
  __syncthreads();
  narrow_turn<D>(Q, tile);
#pragma unroll
  for (int k = 0; k < D * NARROW_CHUNK / 4 / 256; ++k) {
    int i, j;
    narrow_place<D>(p.tall, k, i, j);
    const int r = p.tall ? j0 + j : i, c = p.tall ? i : j0 + j;
    if (r >= res.rows || c >= res.cols) continue;
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = p.tall ? tile[(i + q) * NARROW_PITCH + j] : tile[i * NARROW_PITCH + j + q];
    store_result(res, b, r, c, v);
  }
}

template <class S, int MODE>
int symmetric(const Mats& q, int batch, const float* coef, const Slabs& slabs, int cuts, hipStream_t st) {
  const int t = (q.d + S::BM - 1) / S::BM;
  ALLOW((symmetric_kernel<S, MODE>), S::LDS);
  hipLaunchKernelGGL((symmetric_kernel<S, MODE>), dim3((unsigned)(t * (t + 1) / 2) * batch, cuts), dim3(S::WG_THREADS), S::LDS, st, q, t, coef[0], coef[1], coef[2], slabs);
  if (slabs.out) {
    const int blocks = (int)((q.d * (q.ldg / 8) + 255) / 256);
    hipLaunchKernelGGL(join_kernel, dim3(blocks, batch), dim3(256), 0, st, q, slabs, cuts, S::BM);
  }
  return SGPO_OK;
}
template <class S, bool TALLX, bool LAST>
int apply(const Mats& q, int batch, const Result& r, hipStream_t st) {
  const int tm = (q.rows + S::BM - 1) / S::BM, tn = (q.cols + S::BN - 1) / S::BN;
  ALLOW((apply_kernel<S, TALLX, LAST>), S::LDS);
  hipLaunchKernelGGL((apply_kernel<S, TALLX, LAST>), dim3((unsigned)tm * tn * batch), dim3(S::WG_THREADS), S::LDS, st, q, tm, tn, r);
  return SGPO_OK;
}

// Tile shapes, and what one tile costs (us): `symmetric` and `apply` + `step` per 32 k, `alone` where the tiles are no more than the CUs (of two workgroups
// on a CU one multiplies while the other waits for memory).  Measured at 1 x 1536 x 512, 8 x 512 x 2048, 1024 x 1024, 3 x 400 x 1000 and 16 x 200 x 200.  Small
// tiles spread a small product over the CUs and read more bytes for it; large ones the other way round.  side: odd for the second shape of a side.
struct Kind { int side, per_cu; double symmetric, apply, step, alone; };
constexpr Kind KINDS[] = {{256, 1, 30., 11., 1.40, 1.40}, {192, 1, 17., 9.7, 0.90, 0.90}, {129, 1, 11., 6.4, 0.46, 0.46}, {128, 2, 11., 3.5, 0.575, 0.575},
                          {96, 1, 8.5, 6.8, 0.276, 0.276}, {65, 1, 5.3, 4.2, 0.25, 0.25}, {64, 2, 4.5, 3.6, 0.21, 0.33}, {33, 1, 4.0, 3.7, 0.106, 0.106},
                          {32, 2, 3.6, 3.3, 0.08, 0.147}};
typedef tg::Shape<256, 256, 2, 4, 2, 2> Shape256;
typedef tg::Shape<192, 192, 2, 4, 2, 2> Shape192;
typedef tg::Shape<128, 128, 2, 2, 2, 2, 2> Shape129;   // 128 x 128 with two groups over K: one workgroup fills a CU
typedef tg::Shape<128, 128, 2, 2, 2, 2> Shape128;
typedef tg::Shape<96, 96, 2, 2, 2, 2, 3> Shape96;
typedef tg::Shape<64, 64, 2, 2, 2, 4, 2> Shape65;      // four slots, of which a CU holds one workgroup's: three steps on their way instead of one
typedef tg::Shape<64, 64, 2, 2, 2, 2, 2> Shape64;      // (1024 x 1024: 229 us without, 198 with; four of 768 x 768, more tiles than CUs: 250 without, 296 with)
typedef tg::Shape<32, 32, 1, 1, 2, 4, 4> Shape33;
typedef tg::Shape<32, 32, 1, 1, 2, 2, 4> Shape32;

// The kind with the least rounds of the 256 CUs x cost of a tile; count(side) tiles of `steps` K steps.  A symmetric product with few tiles and a
// long K may also be cut along K (at most `cuts` times), which costs the joining launch and its bytes (two of 150 x 9000, the whole call: 313 us whole, 158 cut).
struct Pick { int kind, cuts; };
template <typename F>
Pick pick(F count, int64_t steps, bool sym, int most_cuts = 1, double joined_bytes = 0.) {
  Pick best = {0, 1};
  double least = 1e300;
  for (int s = 1; s <= most_cuts; s *= 2) {
    if (s > 1 && steps / s < 8) break;
    for (const Kind& k : KINDS) {
      const int64_t n = count(k.side & ~1) * s;
      const double rounds = k.per_cu == 1 ? (double)((n + 255) / 256) : n <= 256 ? 1. : (n + 127) / 128 * 0.5;
      const double t = rounds * ((sym ? k.symmetric : k.apply) + (double)((steps + s - 1) / s) * (n <= 256 ? k.alone : k.step)) + (s > 1 ? 5. + s * joined_bytes * 2. / 4e6 : 0.);
      if (t < least) { least = t; best = {k.side, s}; }
    }
  }
  return best;
}
#define FOR_KIND(K, CALL)                                              \
  switch (K) {                                                         \
    case 256: { typedef Shape256 S; return CALL; }                     \
    case 192: { typedef Shape192 S; return CALL; }                     \
    case 129: { typedef Shape129 S; return CALL; }                     \
    case 128: { typedef Shape128 S; return CALL; }                     \
    case 96: { typedef Shape96 S; return CALL; }                       \
    case 65: { typedef Shape65 S; return CALL; }                       \
    case 64: { typedef Shape64 S; return CALL; }                       \
    case 33: { typedef Shape33 S; return CALL; }                       \
    default: { typedef Shape32 S; return CALL; }                       \
  }
template <int MODE>
int symmetric_any(int kind, const Mats& q, int batch, const float* coef, const Slabs& slabs, int cuts, hipStream_t st) {
  FOR_KIND(kind, (symmetric<S, MODE>(q, batch, coef, slabs, cuts, st)))
}
template <bool TALLX, bool LAST>
int apply_any(int kind, const Mats& q, int batch, const Result& r, hipStream_t st) {
  FOR_KIND(kind, (apply<S, TALLX, LAST>(q, batch, r, st)))
}

constexpr int CUTS = 32;
// Where this takes over from the one launch and from the tiles (us, theirs and this): d <= 32 from 65 on (31 x 128: 31.6, 22.6), d <= 64 from 129 on
// (64 x 128: 39.1, and 64 x 129 41.1 this way), up to 32768 (64 x 32768: 124, 88; the workgroup that adds up the cuts grows with the length's root).
constexpr int NARROW_MOST = 1 << 15;
struct Sizes { int d, longer, narrow, chunks, per, cuts; int64_t ldx, ldg; size_t x, g, off_x, off_y, off_g, off_p, off_s, bytes; Pick gram, poly, full; };
Sizes sizes(int batch, int rows, int cols) {
  Sizes s = {};
  s.d = rows < cols ? rows : cols;
  s.longer = rows < cols ? cols : rows;
  const bool narrow = s.d <= NARROW && s.longer > (s.d <= 32 ? 64 : 128) && s.longer <= NARROW_MOST;
  if (s.longer <= 128 && !narrow) return s;   // one launch, no scratch
  if (narrow) {
    // a cut costs its workgroup a chunk after the other, and the one that adds the cuts up 16 KB of each (64 x 4096: 20 and 32 cuts take the same time)
    s.narrow = s.d <= 32 ? 32 : 64;
    s.chunks = (s.longer + NARROW_CHUNK - 1) / NARROW_CHUNK;
    int64_t cuts = (int64_t)(sqrt(10. * s.chunks) + 1.);
    if (cuts > 1024 / batch) cuts = 1024 / batch;
    if (cuts > s.chunks) cuts = s.chunks;
    if (cuts < 1) cuts = 1;
    s.per = (int)((s.chunks + cuts - 1) / cuts);
    s.cuts = (s.chunks + s.per - 1) / s.per;
    const size_t one = (size_t)batch * s.narrow * s.narrow * 4;
    s.off_g = (size_t)batch * PARTS * 8;
    s.off_s = s.off_g + one;
    s.bytes = s.off_s + one * s.cuts;
    return s;
  }
  s.ldx = round_up(cols, 32) * 2;
  s.ldg = round_up(s.d, 32) * 2;
  s.x = (size_t)rows * s.ldx; s.g = (size_t)s.d * s.ldg;
  size_t at = 0;
  auto take = [&](size_t n) { const size_t o = at; at += (n + 255) & ~(size_t)255; return o; };
  take((size_t)batch * PARTS * 8);
  s.off_x = take(batch * s.x * 2); s.off_y = take(batch * s.x * 2);
  s.off_g = take(batch * s.g * 2); s.off_p = take(batch * s.g * 2);
  auto up = [](int64_t n, int64_t m) { return (n + m - 1) / m; };
  auto triangles = [&](int side) { return batch * up(s.d, side) * (up(s.d, side) + 1) / 2; };
  const double sums = (double)batch * s.d * round_up(s.d, 4) * 4;
  s.gram = pick(triangles, up(s.longer, 32), true, CUTS, sums);
  s.poly = pick(triangles, up(s.d, 32), true);
  s.full = pick([&](int side) { return batch * up(rows, side) * up(cols, side); }, up(s.d, 32), false);
  s.off_s = take(s.gram.cuts > 1 ? (size_t)(s.gram.cuts * sums) : 0);
  s.bytes = at;
  return s;
}

template <typename T, int E>
int orthogonalise_small(const Source& src, int batch, const float* coef, int steps, double eps, const Result& res, hipStream_t st) {
  Table t = {};
  for (int i = 0; i < 3 * steps; ++i) t.v[i] = coef[i];
  ALLOW((small_kernel<T, E>), Small<E>::LDS);
  hipLaunchKernelGGL((small_kernel<T, E>), dim3(batch), dim3(Small<E>::THREADS), Small<E>::LDS, st, src, src.rows < src.cols ? src.rows : src.cols,
                     src.rows < src.cols ? src.cols : src.rows, src.rows > src.cols, t, steps, eps, res);
  SGPO_CHECK_HIP(hipGetLastError());
  return SGPO_OK;
}

template <typename T, int D>
int orthogonalise_narrow(const NarrowArgs& p, int batch, const float* coef, int steps, const Result& res, hipStream_t st) {
  Table t = {};
  for (int i = 0; i < 3 * steps; ++i) t.v[i] = coef[i];
  constexpr int LDS = 4 * D * (D + 4) * 4;
  ALLOW((narrow_poly_kernel<D>), LDS);
  for (int k0 = 0, k1; k0 < steps; k0 = k1) {
    double grown = 1.;
    for (k1 = k0 + 1; k1 < steps; ++k1) {
      const double a = fabs(t.v[3 * k1 - 3]), top = fabs(t.v[3 * k1 - 3] + t.v[3 * k1 - 2] + t.v[3 * k1 - 1]);   // |P| at 0 and at 1
      grown *= a > top ? a * a : top * top;
      if (!(grown < GROWTH)) break;
    }
    if (k0 == 0) hipLaunchKernelGGL((narrow_gram_kernel<T, D, false>), dim3(p.cuts, batch), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((narrow_gram_kernel<T, D, true>), dim3(p.cuts, batch), dim3(256), 0, st, p);
    hipLaunchKernelGGL((narrow_poly_kernel<D>), dim3(batch), dim3(POLY_THREADS<D>), LDS, st, p, t, k0, k1);
  }
  hipLaunchKernelGGL((narrow_apply_kernel<T, D>), dim3(p.chunks, batch), dim3(256), 0, st, p, res);
  SGPO_CHECK_HIP(hipGetLastError());
  return SGPO_OK;
}

template <typename T>
int orthogonalise(Source src, int batch, const float* coef, int steps, double eps, Result res, char* ws, hipStream_t st) {
  const Sizes z = sizes(batch, src.rows, src.cols);
  res.rows = src.rows; res.cols = src.cols;
  if (z.longer <= 64) return orthogonalise_small<T, 64>(src, batch, coef, steps, eps, res, st);
  if (z.longer <= 128 && !z.narrow) return orthogonalise_small<T, 128>(src, batch, coef, steps, eps, res, st);
  double* part = reinterpret_cast<double*>(ws);
  Mats q{(bf16_t*)(ws + z.off_x), (bf16_t*)(ws + z.off_y), (bf16_t*)(ws + z.off_g), (bf16_t*)(ws + z.off_p), z.ldx, z.ldg, (int64_t)z.x, (int64_t)z.g, src.rows, src.cols, z.d};
  const bool tall = src.rows > src.cols;
  src.flat = src.ld == src.cols;
  // about four elements a thread
  const int64_t want = ((int64_t)src.rows * src.cols + 1023) / 1024;
  const int parts = want < PARTS ? (int)want : PARTS;
  hipLaunchKernelGGL((square_kernel<T>), dim3(parts, batch), dim3(256), 0, st, src, part);
  if (z.narrow) {
    const NarrowArgs p{src, part, parts, eps, z.d, z.longer, tall, (float*)(ws + z.off_g), (float*)(ws + z.off_s), z.chunks, z.per, z.cuts};
    return z.narrow == 32 ? orthogonalise_narrow<T, 32>(p, batch, coef, steps, res, st) : orthogonalise_narrow<T, 64>(p, batch, coef, steps, res, st);
  }
  const int64_t blocks = ((int64_t)src.rows * (z.ldx / 8) + 255) / 256;
  // Each workgroup adds up the norm's parts first, so the device is filled once and not more (six 384 x 1536 bf16: 22.3 us with up to 4096 a matrix, 16.1 so).
  const int64_t most = batch < 32 ? 2048 / batch : 64;
  hipLaunchKernelGGL((load_kernel<T>), dim3((unsigned)(blocks < most ? blocks : most), batch), dim3(256), 0, st, src, part, parts, eps, q.X, z.ldx, (int64_t)z.x);
  Slabs slabs = {nullptr, 0, 0};
  int cuts = 1;
  if (z.gram.cuts > 1) {
    const int steps_k = (z.longer + 31) / 32, per = (steps_k + z.gram.cuts - 1) / z.gram.cuts;
    cuts = (steps_k + per - 1) / per;
    slabs = Slabs{(float*)(ws + z.off_s), per, (int)round_up(z.d, 4)};
  }
  const int kg = z.gram.kind, kp = z.poly.kind, ka = z.full.kind;
  for (int k = 0; k < steps; ++k) {
    int rc = tall ? symmetric_any<TALL>(kg, q, batch, coef + 3 * k, slabs, cuts, st) : symmetric_any<WIDE>(kg, q, batch, coef + 3 * k, slabs, cuts, st);
    if (!rc) rc = symmetric_any<POLY>(kp, q, batch, coef + 3 * k, Slabs{nullptr, 0, 0}, 1, st);
    if (!rc) {
      if (k + 1 < steps) rc = tall ? apply_any<true, false>(ka, q, batch, res, st) : apply_any<false, false>(ka, q, batch, res, st);
      else rc = tall ? apply_any<true, true>(ka, q, batch, res, st) : apply_any<false, true>(ka, q, batch, res, st);
    }
    if (rc) return rc;
    bf16_t* t = q.X; q.X = q.Y; q.Y = t;
  }
  SGPO_CHECK_HIP(hipGetLastError());
  return SGPO_OK;
}

constexpr int MOST = 1 << 22;
bool overlap(const void* a, int64_t na, const void* b, int64_t nb) { return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na; }   // bytes

int check_sizes(int batch, int rows, int cols, int steps, const float* coef) {
  SGPO_REQUIRE(batch >= 0 && rows >= 0 && cols >= 0, "newton_schulz: negative size");
  SGPO_REQUIRE(batch <= 65535 && (int64_t)rows * cols <= 0x7fffffff && (int64_t)batch * rows * cols <= ((int64_t)1 << 40), "newton_schulz: %d matrices of %d x %d over the supported range",
               batch, rows, cols);
  // 256 rows of X, two planes each, lie within the 32-bit offsets of the tiles' loads
  SGPO_REQUIRE(rows <= MOST && cols <= MOST, "newton_schulz: %d x %d: at most %d rows or columns", rows, cols, MOST);
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
  SGPO_REQUIRE(update && out, "newton_schulz: null argument");
  SGPO_REQUIRE(ld >= cols || rows == 1, "newton_schulz: row pitch %lld below %d columns", (long long)ld, cols);
  const size_t need = sgpo_newton_schulz_workspace_bytes(batch, rows, cols);
  SGPO_REQUIRE((uintptr_t)workspace % 256 == 0, "newton_schulz: the workspace must be 256-byte aligned");
  if (need && (!workspace || workspace_bytes < need)) { sgpo_set_error("newton_schulz: workspace %zu < %zu", workspace_bytes, need); return SGPO_ERR_WORKSPACE; }
  const int esz = dtype == SGPO_DTYPE_BF16 ? 2 : 4;
  SGPO_REQUIRE(stride_b >= 0 && !overlap(update, ((batch - 1) * stride_b + (rows - 1) * ld + cols) * esz, out, (int64_t)batch * rows * cols * 2), "newton_schulz: out overlaps update");
  const Source s{update, nullptr, 0.f, 0, stride_b, ld, rows, cols, 0};
  const Result r{out, 1, 0, 0, 0, 0.f, 0.f};
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
  SGPO_REQUIRE(weight && grad && momentum_buffer, "muon_step: null argument");
  const size_t need = sgpo_newton_schulz_workspace_bytes(batch, rows, cols);
  SGPO_REQUIRE((uintptr_t)workspace % 256 == 0, "muon_step: the workspace must be 256-byte aligned");
  if (need && (!workspace || workspace_bytes < need)) { sgpo_set_error("muon_step: workspace %zu < %zu", workspace_bytes, need); return SGPO_ERR_WORKSPACE; }
  const int64_t n = (int64_t)batch * rows * cols, wb = n * (weight_dtype == SGPO_DTYPE_BF16 ? 2 : 4), gb = n * (grad_dtype == SGPO_DTYPE_BF16 ? 2 : 4);
  SGPO_REQUIRE(!overlap(weight, wb, grad, gb) && !overlap(weight, wb, momentum_buffer, n * 4) && !overlap(grad, gb, momentum_buffer, n * 4),
               "muon_step: weight, grad and momentum_buffer overlap");
  const Source s{grad, momentum_buffer, momentum, nesterov != 0, (int64_t)rows * cols, cols, rows, cols, 0};
  const double ratio = rows > cols ? (double)rows / cols : 1.0;
  const Result r{weight, weight_dtype == SGPO_DTYPE_BF16, 0, 0, 1, (float)(1.0 - (double)lr * weight_decay), (float)(lr * sqrt(ratio))};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return grad_dtype == SGPO_DTYPE_BF16 ? orthogonalise<bf16_t>(s, batch, coefficients, steps, eps, r, (char*)workspace, st)
                                       : orthogonalise<float>(s, batch, coefficients, steps, eps, r, (char*)workspace, st);
}
