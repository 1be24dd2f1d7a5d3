// Cross entropy of a linear vocabulary head without its logits.
//
//   z = hidden weight^T + bias          [N][V], never stored
//   lse_i = log sum_v exp z_iv          nll_i = lse_i - z_i,t(i)          (0 where t(i) = ignore_index)
//   d_iv = g_i (exp(z_iv - lse_i) - [v = t(i)])      dhidden = d weight,  dweight = d^T hidden,  dbias = sum_i d_iv
//
// Forward: one pass of output tiles over (tokens, classes).  A tile leaves its logits in the accumulators and writes one
// (maximum, sum of exponentials) pair per token; a second kernel joins a token's pairs.  Backward: the vocabulary in pieces;
// for each piece the logits again, d (rounded to the operands' precision) into a buffer that every piece reuses, then the two products
// that read it -- d as rows (dhidden) and d as columns (dweight) come from the same buffer (tile_gemm.h, KC and KM).
// 2 N V H operations forward and 6 backward.  Logits stay in registers; a piece of d goes through memory: 8192 tokens by 16384 classes of bf16 are 256 MB
// written, and each of the two products reads about three times that, operands included (770 and 830 MB in 0.41 ms, 2.1 TB/s).
//
// bf16 operands: one plane; d is rounded to bf16 once (2^-8 of a term at most, of the size of the outputs' own rounding), sums in
// fp32.  A factor common to all tokens (mean, sum) is left out of d and applied to the products' sums: rounded into d it would be off
// by the same up to 2^-8 everywhere, while p - 1 of an unlikely target is -1 almost exactly.  fp32 operands: three planes, i.e. products and d with 24 bits.
// Sums over tokens and classes run in a fixed order: the same inputs give the same bits.
#include "../../include/sgpo_hip.h"
#include "tile_gemm.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

__host__ __device__ inline int64_t round_up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

// ------------------------------------------------------------------------------------------------ operands as planes
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<bf16_t>(bf16_t v) { return bf2f(v); }

// dst [rows_out][cols_out] planes, zero beyond src's rows x cols and in rows whose target is ignore_index (their features may be
// anything, and 0 * inf is no 0)
template <typename T, int PL>
__global__ __launch_bounds__(256) void pack_kernel(const T* src, int64_t ld, int rows, int cols, bf16_t* dst, int64_t rows_out,
                                                   int cols_out, const int64_t* targets, int64_t ignore) {
  const int quads = cols_out >> 2;
  const int64_t total = rows_out * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / quads;
    const int e = (int)(i - r * quads) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < rows && !(targets && targets[r] == ignore)) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (e + q < cols) v[q] = to_f32<T>(src[r * ld + e + q]);
    }
    tg::store4<PL>(dst + r * (int64_t)cols_out * PL, e, v);
  }
}

// dst [cols_out][rows_out] = src transposed, bf16, with the same zeros; 64 x 64 tiles through LDS
__global__ __launch_bounds__(256) void transpose_kernel(const bf16_t* src, int64_t ld, int rows, int cols, bf16_t* dst, int64_t rows_out,
                                                        const int64_t* targets, int64_t ignore) {
  __shared__ bf16_t tile[64][66];
  const int64_t r0 = (int64_t)blockIdx.x * 64;
  const int c0 = blockIdx.y * 64;
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int r = i >> 6, c = i & 63;
    const bool in = r0 + r < rows && c0 + c < cols && targets[r0 + r] != ignore;
    tile[c][r] = in ? src[(r0 + r) * ld + c0 + c] : (bf16_t)0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * 32; i += 256) {
    const int c = i >> 5, r = (i & 31) * 2;
    *reinterpret_cast<uint32_t*>(dst + (int64_t)(c0 + c) * rows_out + r0 + r) = *reinterpret_cast<const uint32_t*>(&tile[c][r]);
  }
}

// ------------------------------------------------------------------------------------------------------------ forward
struct LossArgs {
  tg::Operand h, w;
  const float* bias;        // [V] or null; -inf closes a class
  const int64_t* targets;
  int64_t ignore;
  int r0, n_rows;           // rows [r0, r0 + n_rows) of the tokens
  int v0, n_cls;            // classes [v0, v0 + n_cls)
  int nk;
};

template <class S>
__device__ __forceinline__ void logits(const LossArgs& p, int m0, int n0, char* smem, f32x4 (&acc)[S::MT][S::NT]) {
  tg::clear<S>(acc);
  tg::run<S, tg::KC, tg::KC>(p.h, p.w, m0, n0, 0, p.nk, smem, acc);
  const int lane = threadIdx.x & 63, l4 = lane >> 4;
  const int wave = (int)threadIdx.x >> 6, wn = wave % S::WN;
  const int c0 = n0 + wn * S::NT * 16 + 4 * l4;
  if (p.bias) {
#pragma unroll
    for (int y = 0; y < S::NT; ++y)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float b = p.bias[p.v0 + min(c0 + y * 16 + q, p.n_cls - 1)];
#pragma unroll
        for (int x = 0; x < S::MT; ++x) acc[x][y][q] += b;
      }
  }
  if (n0 + S::BN > p.n_cls) {   // the last column of tiles: classes that do not exist
#pragma unroll
    for (int y = 0; y < S::NT; ++y)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (c0 + y * 16 + q >= p.n_cls) {
#pragma unroll
          for (int x = 0; x < S::MT; ++x) acc[x][y][q] = -INFINITY;
        }
  }
}

__device__ __forceinline__ float lanes4_max(float v) {   // over the four lanes that share l16
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float lanes4_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
// (m, s) of a union from two (maximum, sum of exp(z - maximum)) pairs; empty is (-inf, 0), NaN travels in s
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.f : top;
  s = s * __builtin_amdgcn_exp2f((m - ref) * LOG2E) + s2 * __builtin_amdgcn_exp2f((m2 - ref) * LOG2E);
  m = top;
}

__device__ __forceinline__ void store_loss(float l, float at_target, int64_t t, int64_t ignore, int V, float* nll, float* lse) {
  *lse = l;
  // a target that is no class has no loss: NaN, so that the step shows it
  *nll = t == ignore ? 0.f : (t < 0 || t >= V) ? __builtin_nanf("") : l - at_target;
}

// part[tile column][row of the chunk] = (max, sum);  at_target[row] = the target's logit
template <class S>
__global__ __launch_bounds__(S::THREADS, 2) void lse_kernel(LossArgs p, int tm, int tn, float2* part, float* at_target) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int im, in;
  tg::tile_of(blockIdx.x, tm, tn, im, in);
  const int m0 = im * S::BM, n0 = in * S::BN;
  f32x4 acc[S::MT][S::NT];
  logits<S>(p, m0, n0, smem, acc);
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = (int)threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  float2* share = reinterpret_cast<float2*>(smem);   // [WN][BM]
#pragma unroll
  for (int x = 0; x < S::MT; ++x) {
    const int lm = (wm * S::MT + x) * 16 + l16, m = m0 + lm;
    float top = -INFINITY;
#pragma unroll
    for (int y = 0; y < S::NT; ++y)
#pragma unroll
      for (int q = 0; q < 4; ++q) top = fmaxf(top, acc[x][y][q]);
    top = lanes4_max(top);
    const float ref = top == -INFINITY ? 0.f : top;
    float s = 0.f;
#pragma unroll
    for (int y = 0; y < S::NT; ++y)
#pragma unroll
      for (int q = 0; q < 4; ++q) s += __builtin_amdgcn_exp2f((acc[x][y][q] - ref) * LOG2E);
    s = lanes4_sum(s);
    if (l4 == 0) share[wn * S::BM + lm] = make_float2(top, s);
    if (m < p.n_rows) {
      const int64_t t = p.targets[p.r0 + m] - p.v0;
      const int64_t tq = t - n0 - wn * S::NT * 16 - 4 * l4;   // 16 y + q, if the class lies with this lane
      if (tq >= 0 && tq < S::NT * 16 && (tq & 12) == 0 && t < p.n_cls) {
#pragma unroll
        for (int y = 0; y < S::NT; ++y)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (16 * y + q == (int)tq) at_target[m] = acc[x][y][q];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < S::BM; i += S::THREADS) {
    float2 a = share[i];
#pragma unroll
    for (int w = 1; w < S::WN; ++w) {
      const float2 b = share[w * S::BM + i];
      join(a.x, a.y, b.x, b.y);
    }
    if (m0 + i < p.n_rows) part[(int64_t)in * p.n_rows + m0 + i] = a;
  }
}

// joins a token's pairs: 16 tokens per workgroup, 16 threads share a token's tile columns
__global__ __launch_bounds__(256) void finish_kernel(const float2* part, int n_rows, int tn, const float* at_target, const int64_t* targets,
                                                     int64_t ignore, int V, float* nll, float* lse) {
  __shared__ float2 share[16][17];
  const int r = threadIdx.x & 15, w = threadIdx.x >> 4;
  const int m = blockIdx.x * 16 + r;
  float a = -INFINITY, s = 0.f;
  if (m < n_rows)
    for (int i = w; i < tn; i += 16) {
      const float2 b = part[(int64_t)i * n_rows + m];
      join(a, s, b.x, b.y);
    }
  share[w][r] = make_float2(a, s);
  __syncthreads();
  if (w == 0 && m < n_rows) {
#pragma unroll
    for (int i = 1; i < 16; ++i) join(a, s, share[i][r].x, share[i][r].y);
    store_loss(a + logf(s), at_target[m], targets[m], ignore, V, nll + m, lse + m);
  }
}

// loss[0] = sum of nll (reduction 2) or its mean over the tokens with a loss (1; 0 if there are none); inv[0] = the factor on every token's gradient,
// 0 if none has one.
// Over TOTAL_ROWS tokens a workgroup to as many writes its part and one more adds the parts up (65536 tokens: 8.3 us; by one workgroup 20.6).
constexpr int TOTAL_ROWS = 8192;
struct Part { double sum; int64_t count; };
__device__ __forceinline__ Part block_total(double s, int64_t c) {   // valid in thread 0
  __shared__ double ssum[16];
  __shared__ int64_t scnt[16];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { s += __shfl_xor(s, o); c += __shfl_xor(c, o); }
  if ((threadIdx.x & 63) == 0) { ssum[threadIdx.x >> 6] = s; scnt[threadIdx.x >> 6] = c; }
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 1; i < 16; ++i) { s += ssum[i]; c += scnt[i]; }
  return Part{s, c};
}
__device__ __forceinline__ Part rows_total(const float* nll, const int64_t* targets, int64_t ignore, int64_t first, int n) {
  double s = 0.0;
  int64_t c = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += 1024) {
    s += (double)nll[first + i];
    c += targets[first + i] != ignore;
  }
  return block_total(s, c);
}
__device__ __forceinline__ void store_total(const Part& p, int mean, float* loss, float* inv) {
  const double n = mean ? (double)(p.count > 0 ? p.count : 1) : 1.0;
  loss[0] = (float)(p.sum / n);
  inv[0] = p.count > 0 ? (float)(1.0 / n) : 0.f;
}
__global__ __launch_bounds__(1024) void total_kernel(const float* nll, const int64_t* targets, int64_t ignore, int N, int mean, float* loss, float* inv) {
  const Part p = rows_total(nll, targets, ignore, 0, N);
  if (threadIdx.x == 0) store_total(p, mean, loss, inv);
}
__global__ __launch_bounds__(1024) void parts_kernel(const float* nll, const int64_t* targets, int64_t ignore, int N, Part* parts) {
  const int64_t first = (int64_t)blockIdx.x * TOTAL_ROWS;
  const Part p = rows_total(nll, targets, ignore, first, (int)min((int64_t)TOTAL_ROWS, N - first));
  if (threadIdx.x == 0) parts[blockIdx.x] = p;
}
__global__ __launch_bounds__(1024) void join_total_kernel(const Part* parts, int n, int mean, float* loss, float* inv) {
  double s = 0.0;
  int64_t c = 0;
  for (int i = threadIdx.x; i < n; i += 1024) { s += parts[i].sum; c += parts[i].count; }
  const Part p = block_total(s, c);
  if (threadIdx.x == 0) store_total(p, mean, loss, inv);
}

// ----------------------------------------------------------------------------------------------------------- backward
// The factor common to all tokens' gradients; 1 where each has its own.  No token with a loss: 0, whatever the upstream gradient is.
struct Factor {
  const float *g, *inv;   // null: 1
  __device__ __forceinline__ float get() const {
    if (!g) return 1.f;
    const float up = g[0], i = inv[0];   // both on their way at once
    return i == 0.f ? 0.f : up * i;
  }
};

// d (without the common factor) of a piece of the vocabulary into d [rows_pad][cols_pad] planes (zero beyond the tokens and classes); column sums per row tile
template <class S>
__global__ __launch_bounds__(S::THREADS, 2) void grad_kernel(LossArgs p, int tm, int tn, const float* lse, const float* g,
                                                               int g_rows, bf16_t* d, int rows_pad, int cols_pad,
                                                               float* col_sums) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int im, in;
  tg::tile_of(blockIdx.x, tm, tn, im, in);
  const int m0 = im * S::BM, n0 = in * S::BN;
  f32x4 acc[S::MT][S::NT];
  logits<S>(p, m0, n0, smem, acc);
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = (int)threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  float cs[S::NT][4];
#pragma unroll
  for (int y = 0; y < S::NT; ++y)
#pragma unroll
    for (int q = 0; q < 4; ++q) cs[y][q] = 0.f;
  // The planes of XG row blocks at a time pass through this wave's part of the LDS, so that they leave in whole lines: from the registers a
  // row would go out in pieces of 32 bytes (a piece of 8192 x 16384: 610 us with those, 506 so).
  constexpr int RB = S::NT * 32 * S::PL, CH = RB / 16, MASK = CH % 8 == 0 ? 7 : 3;   // bytes and 16-B chunks of a wave's row
  constexpr int PART = S::LDS / (S::WM * S::WN), FIT = PART / (16 * RB), XG = FIT >= S::MT ? S::MT : FIT >= S::MT / 2 ? S::MT / 2 : 1;
  static_assert(XG * 16 * RB <= PART && S::MT % XG == 0, "a row block fits the wave's part");
  char* mine = smem + wave * PART;
  const int nb = n0 + wn * S::NT * 16;   // the wave's first column
#pragma unroll
  for (int g0 = 0; g0 < S::MT; g0 += XG) {
#pragma unroll
    for (int xx = 0; xx < XG; ++xx) {
      const int x = g0 + xx, m = m0 + (wm * S::MT + x) * 16 + l16;
      const bool in_rows = m < p.n_rows;
      const int64_t t = in_rows ? p.targets[m] : p.ignore;
      const bool keep = in_rows && t != p.ignore;
      const bool bad = keep && (t < 0 || t >= (int64_t)p.w.rows + p.v0);
      const float l = keep ? lse[m] : 0.f;
      const float gm = keep ? (bad ? __builtin_nanf("") : g_rows ? g[m] : 1.f) : 0.f;
      const int64_t tw = t - p.v0 - nb - 4 * l4;
      const int tq = tw >= 0 && tw < S::NT * 16 ? (int)tw : -1;   // 16 y + q, if the class lies with this lane
#pragma unroll
      for (int y = 0; y < S::NT; ++y) {
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float e = __builtin_amdgcn_exp2f((acc[x][y][q] - l) * LOG2E);
          v[q] = gm * (16 * y + q == tq ? e - 1.f : e);
          v[q] = keep ? v[q] : 0.f;
          cs[y][q] += v[q];
        }
        float pl[4][S::PL];
#pragma unroll
        for (int q = 0; q < 4; ++q) tg::split<S::PL>(v[q], pl[q]);
        const int r = xx * 16 + l16, e0 = y * 16 + 4 * l4;   // element within the wave's row
#pragma unroll
        for (int k = 0; k < S::PL; ++k) {
          const int at = (e0 >> 5) * (64 * S::PL) + k * 64 + (e0 & 31) * 2;   // bytes
          *reinterpret_cast<uint2*>(mine + r * RB + (((at >> 4) ^ (r & MASK)) << 4) + (at & 15)) =
              make_uint2(pack_bf16x2(pl[0][k], pl[1][k]), pack_bf16x2(pl[2][k], pl[3][k]));
        }
      }
    }
    __builtin_amdgcn_wave_barrier();   // one wave's LDS accesses run in order: nothing to wait for but the data
#pragma unroll 4
    for (int i = lane; i < XG * 16 * CH; i += 64) {
      const int r = i / CH, c = i - r * CH, m = m0 + (wm * S::MT + g0) * 16 + r;
      const uint4 v = *reinterpret_cast<const uint4*>(mine + r * RB + ((c ^ (r & MASK)) << 4));
      if (m < rows_pad && nb < cols_pad)
        *reinterpret_cast<uint4*>(reinterpret_cast<char*>(d + ((int64_t)m * cols_pad + nb) * S::PL) + c * 16) = v;
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (!col_sums) return;
  __syncthreads();
  float* share = reinterpret_cast<float*>(smem);   // [WM][BN]
#pragma unroll
  for (int y = 0; y < S::NT; ++y)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float s = cs[y][q];
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) s += __shfl_xor(s, o);
      if (l16 == 0) share[wm * S::BN + (wn * S::NT + y) * 16 + 4 * l4 + q] = s;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < S::BN; i += S::THREADS) {
    float s = share[i];
#pragma unroll
    for (int w = 1; w < S::WM; ++w) s += share[w * S::BN + i];
    if (n0 + i < p.n_cls) col_sums[(int64_t)im * p.n_cls + n0 + i] = s;
  }
}

// ------------------------------------------------------------------------------------ small vocabularies (up to 64 classes)
// A head of at most 64 classes is bound by reading the features.  A wave takes 16 tokens and all classes; operands go from memory straight
// into fragments (fp32 ones are cut into planes in registers), so there is no LDS staging, no packed copy and, all of a token's
// classes being in one wave, no second kernel.  KS = 4: the four waves of a workgroup share the features of 16 tokens (few tokens: four times the
// workgroups and a quarter of the chain), KS = 1: 16 tokens each.
// GRAD: d instead of the loss, and on the way the packed copy of the features that dweight's product reads.
struct HeadArgs {
  const void *h, *w;
  int64_t ldh, ldw;
  const float* bias;
  const int64_t* targets;
  int64_t ignore;
  int N, H, V;
  float *nll, *lse;          // forward's outputs; GRAD reads lse
  const float* g;            // [N], or not read (g_rows 0)
  int g_rows, rows_pad, h_pad;
  bf16_t *d, *hp;            // [rows_pad][64], [rows_pad][h_pad] planes
  float* col_sums;           // [workgroup][V], or null
};
inline int head_rows(int64_t N) { return N <= 8192 ? 16 : 64; }   // tokens of a workgroup; few tokens: four waves to 16 of them

template <typename T> struct PlanesOf { static constexpr int value = 1; };
template <> struct PlanesOf<float> { static constexpr int value = 3; };

// eight consecutive features of a row as fragments of each plane, zero from `limit` on; rows need no more than their elements' alignment
template <typename T, int PL>
__device__ __forceinline__ void load8(const T* row, int e, int limit, bool live, bf16x8 (&f)[PL]) {
  alignas(16) T x[8];
  if (e + 8 <= limit) {
    __builtin_memcpy(x, row + e, sizeof(x));   // 16-byte loads, also of odd rows (56377 x 1143 bf16, 31 classes: 338 us element by element, 109 so)
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = e + i < limit ? row[e + i] : T(0);
  }
  if constexpr (PL == 1) {
    f[0] = live ? *reinterpret_cast<const bf16x8*>(x) : bf16x8{};
  } else {
    uint32_t w[PL][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float p0[PL], p1[PL];
      tg::split<PL>(live ? x[2 * i] : 0.f, p0);
      tg::split<PL>(live ? x[2 * i + 1] : 0.f, p1);
#pragma unroll
      for (int p = 0; p < PL; ++p) w[p][i] = pack_bf16x2(p0[p], p1[p]);
    }
#pragma unroll
    for (int p = 0; p < PL; ++p) f[p] = *reinterpret_cast<const bf16x8*>(&w[p]);
  }
}

template <typename T, int NB, int KS, bool GRAD>
__global__ __launch_bounds__(256) void head_kernel(HeadArgs p) {
  constexpr int PL = PlanesOf<T>::value;
  __shared__ f32x4 share[KS > 1 ? KS - 1 : 1][NB][64];
  __shared__ float sums[KS > 1 ? 1 : 4][64];
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), ks = KS > 1 ? wave : 0;
  const int m = ((int)blockIdx.x * (4 / KS) + (KS > 1 ? 0 : wave)) * 16 + l16;
  const int64_t t = m < p.N ? p.targets[m] : p.ignore;
  const bool keep = m < p.N && t != p.ignore;
  const T* hr = reinterpret_cast<const T*>(p.h) + (int64_t)min(m, p.N - 1) * p.ldh;
  const T* wr[NB];
#pragma unroll
  for (int y = 0; y < NB; ++y) wr[y] = reinterpret_cast<const T*>(p.w) + (int64_t)min(y * 16 + l16, p.V - 1) * p.ldw;
  f32x4 acc[NB];
#pragma unroll
  for (int y = 0; y < NB; ++y) acc[y] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int H = p.H, slices = (H + 31) >> 5;
  auto slice = [&](int s, int limit) {   // limit: H, or no limit for whole slices
    const int e = s * 32 + l4 * 8;
    bf16x8 a[PL], b[NB][PL];
    load8<T, PL>(hr, e, limit, GRAD ? keep : true, a);
#pragma unroll
    for (int y = 0; y < NB; ++y) load8<T, PL>(wr[y], e, limit, true, b[y]);
    if constexpr (GRAD) {
      if (p.hp && m < p.rows_pad) {
#pragma unroll
        for (int q = 0; q < PL; ++q) *reinterpret_cast<bf16x8*>(p.hp + (int64_t)m * p.h_pad * PL + s * 32 * PL + q * 32 + l4 * 8) = a[q];
      }
    }
#pragma unroll
    for (int i = 0; i < PL; ++i)
#pragma unroll
      for (int j = 0; i + j < PL; ++j)
#pragma unroll
        for (int y = 0; y < NB; ++y) acc[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[y][j], a[i], acc[y], 0, 0, 0);
  };
  int s = ks;
  for (; (s + 1) * 32 <= H; s += KS) slice(s, INT_MAX);
  for (; s < slices; s += KS) slice(s, H);
  if constexpr (GRAD) {   // the packed features' last padding
    const int ps = p.h_pad >> 5;
    for (; s < ps; s += KS)
      if (p.hp && m < p.rows_pad)
#pragma unroll
        for (int q = 0; q < PL; ++q) *reinterpret_cast<bf16x8*>(p.hp + (int64_t)m * p.h_pad * PL + s * 32 * PL + q * 32 + l4 * 8) = bf16x8{};
  }
  if constexpr (KS > 1) {
    if (ks > 0)
#pragma unroll
      for (int y = 0; y < NB; ++y) share[ks - 1][y][lane] = acc[y];
    __syncthreads();
    if (ks > 0) return;
#pragma unroll
    for (int k = 1; k < KS; ++k)
#pragma unroll
      for (int y = 0; y < NB; ++y) acc[y] += share[k - 1][y][lane];
  }
  float top = -INFINITY, at = 0.f;
  const bool cls = t >= 0 && t < p.V;
#pragma unroll
  for (int y = 0; y < NB; ++y)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = y * 16 + 4 * l4 + q;
      const bool in = n < p.V;
      const float z = in ? acc[y][q] + (p.bias ? p.bias[n] : 0.f) : -INFINITY;
      acc[y][q] = z;
      top = fmaxf(top, z);
      if (cls && n == (int)t) at = z;
    }
  if constexpr (!GRAD) {
    top = lanes4_max(top);
    at = lanes4_sum(at);   // three of the four lanes hold 0
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int q = 0; q < 4; ++q) sum += __builtin_amdgcn_exp2f((acc[y][q] - ref) * LOG2E);
    sum = lanes4_sum(sum);
    if (l4 == 0 && m < p.N) store_loss(top + logf(sum), at, t, p.ignore, p.V, p.nll + m, p.lse + m);
  } else {
    const float l = keep ? p.lse[m] : 0.f;
    const float gm = keep ? (cls ? (p.g_rows ? p.g[m] : 1.f) : __builtin_nanf("")) : 0.f;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int n = y * 16 + 4 * l4;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (y < NB) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float e = __builtin_amdgcn_exp2f((acc[y < NB ? y : 0][q] - l) * LOG2E);
          v[q] = keep && n + q < p.V ? gm * (e - (cls && n + q == (int)t ? 1.f : 0.f)) : 0.f;
        }
      }
      if (m < p.rows_pad) tg::store4<PL>(p.d + (int64_t)m * 64 * PL, n, v);
      if (p.col_sums && y < NB) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
          for (int o = 1; o < 16; o <<= 1) v[q] += __shfl_xor(v[q], o);
          if (l16 == 0) {
            if constexpr (KS > 1) { if (n + q < p.V) p.col_sums[(int64_t)blockIdx.x * p.V + n + q] = v[q]; }
            else sums[wave][n + q] = v[q];
          }
        }
      }
    }
    if constexpr (KS == 1) {
      if (!p.col_sums) return;
      __syncthreads();
      const int n = threadIdx.x;
      if (n < p.V) p.col_sums[(int64_t)blockIdx.x * p.V + n] = (sums[0][n] + sums[1][n]) + (sums[2][n] + sums[3][n]);
    }
  }
}

// C tile of a product, K split over gridDim.y slabs: fp32 (added to what is there if `add`) or rounded to bf16
struct MmArgs {
  tg::Operand a, b;
  int M, N, nk, nk_split;
  void* out;
  int64_t ldo, slab;
  Factor factor;            // on the sums
  const int64_t* targets;   // or null: rows whose target is ignore get the factor 0 (an infinite one would make their zeros NaN)
  int64_t ignore;
  int out_bf16, add;
};

template <class S, int KA, int KB>
__global__ __launch_bounds__(S::WG_THREADS, 2) void mm_kernel(MmArgs p, int tm, int tn) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int im, in;
  tg::tile_of(blockIdx.x, tm, tn, im, in);
  const int m0 = im * S::BM, n0 = in * S::BN;
  const int k0 = blockIdx.y * p.nk_split, nk = min(p.nk_split, p.nk - k0);
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wm = S::wave() / S::WN, wn = S::wave() % S::WN;
  int64_t target[S::MT];   // of all rows, on their way during the products
#pragma unroll
  for (int x = 0; x < S::MT; ++x) target[x] = p.targets ? p.targets[min(m0 + (wm * S::MT + x) * 16 + l16, p.M - 1)] : 0;
  f32x4 acc[S::MT][S::NT];
  tg::clear<S>(acc);
  tg::run<S, KA, KB>(p.a, p.b, m0, n0, k0, nk, smem, acc);
  const float factor = p.factor.get();
#pragma unroll
  for (int x = 0; x < S::MT; ++x) {
    const int m = m0 + (wm * S::MT + x) * 16 + l16;
    if (m >= p.M) continue;
    const float f = p.targets && target[x] == p.ignore ? 0.f : factor;
#pragma unroll
    for (int y = 0; y < S::NT; ++y) {
      if (!S::owns(x, y)) continue;
      const int n = n0 + (wn * S::NT + y) * 16 + 4 * l4;
      f32x4 v = acc[x][y] * f;
      // four at a time, whatever the row's alignment (dhidden of 56377 x 1143 bf16, 31 classes: 109 us element by element, 49 so)
      if (p.out_bf16) {
        bf16_t* o = reinterpret_cast<bf16_t*>(p.out) + m * p.ldo + n;
        const uint32_t w[2] = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        if (n + 4 <= p.N) __builtin_memcpy(o, w, 8);
        else
#pragma unroll
          for (int q = 0; q < 4; ++q) if (n + q < p.N) o[q] = f2bf(v[q]);
      } else {
        float* o = reinterpret_cast<float*>(p.out) + blockIdx.y * p.slab + m * p.ldo + n;
        if (n + 4 <= p.N) {
          if (p.add) {
            f32x4 was;
            __builtin_memcpy(&was, o, 16);
            v += was;
          }
          __builtin_memcpy(o, &v, 16);
        } else
#pragma unroll
          for (int q = 0; q < 4; ++q) if (n + q < p.N) o[q] = p.add ? o[q] + v[q] : v[q];
      }
    }
  }
}

// out[r][c] = sum over slabs of src[slab][r][c], up to three such sums in a launch.  `spread` threads share an output's slabs (few outputs of
// many slabs would leave the card to a chain of loads) and add up in a fixed order.
struct SumJob {
  const float* src;
  void* out;
  int64_t slab, ld, total;   // ld: src's row pitch; total = rows * cols
  int n_slabs, cols, out_bf16, spread, blocks;
  Factor factor;
};
struct SumJobs { SumJob j[3]; };
__global__ __launch_bounds__(256) void sum_kernel(SumJobs jobs) {
  __shared__ float share[256];
  int b = blockIdx.x, k = 0;
  while (k < 2 && b >= jobs.j[k].blocks) b -= jobs.j[k++].blocks;
  const SumJob& p = jobs.j[k];
  const int per = 256 / p.spread, o = threadIdx.x % per, g = threadIdx.x / per;
  for (int64_t i0 = (int64_t)b * per; i0 < p.total; i0 += (int64_t)p.blocks * per) {
    const int64_t i = i0 + o;
    float s = 0.f;
    if (i < p.total) {
      const int64_t r = p.total >> 32 ? i / p.cols : (uint32_t)i / (uint32_t)p.cols;
      const float* src = p.src + r * p.ld + (i - r * p.cols);
#pragma unroll 8
      for (int k2 = g; k2 < p.n_slabs; k2 += p.spread) s += src[k2 * p.slab];
    }
    if (p.spread > 1) {
      __syncthreads();
      share[threadIdx.x] = s;
      __syncthreads();
      if (g == 0)
        for (int q = 1; q < p.spread; ++q) s += share[q * per + o];
    }
    if (g == 0 && i < p.total) {
      s *= p.factor.get();
      if (p.out_bf16) reinterpret_cast<bf16_t*>(p.out)[i] = f2bf(s);
      else reinterpret_cast<float*>(p.out)[i] = s;
    }
  }
}

__global__ __launch_bounds__(256) void fill_kernel(float* p, int64_t n, float v) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = v;
}

// ---------------------------------------------------------------------------------------------------------- host side
// Tile shapes by planes: L, M, S for the kernels that reduce over a tile's rows, and for the products P (S with two groups over K).
template <int PL> struct Shapes;
template <> struct Shapes<1> {
  typedef tg::Shape<256, 256, 2, 4, 1, 2> L;
  typedef tg::Shape<128, 128, 2, 2, 1, 2> M;
  typedef tg::Shape<64, 64, 2, 2, 1, 4> S;
  typedef tg::Shape<64, 64, 2, 2, 1, 2, 2> P;
};
template <> struct Shapes<3> {
  typedef tg::Shape<256, 128, 4, 2, 3, 2> L;
  typedef tg::Shape<128, 128, 2, 4, 3, 2> M;
  typedef tg::Shape<64, 64, 2, 2, 3, 2> S;
  typedef tg::Shape<64, 64, 2, 2, 3, 2, 2> P;
};
int config_bn(int PL, int c) { return PL == 1 ? (c == 2 ? 256 : c == 1 ? 128 : 64) : (c ? 128 : 64); }
int config_bm(int PL, int c) { return c == 2 ? 256 : c == 1 ? 128 : 64; }

inline int64_t tiles(int64_t m, int64_t n, int bm, int bn) { return (m + bm - 1) / bm * ((n + bn - 1) / bn); }

// the largest tile that still gives most of the CUs one
int pick(int PL, int64_t M, int64_t N) {
  for (int c = 2; c > 0; --c)
    if (tiles(M, N, config_bm(PL, c), config_bn(PL, c)) >= 160) return c;
  return 0;
}

// A product's tile shape and the slabs its K is cut into: the least of the CUs' rounds x (fixed + steps x step), and the slabs' sum.  A step costs
// a workgroup of the smaller shapes less than twice as much where two share a CU: alone, it waits for memory.  Costs of one tile in us,
// fitted to 138 products of 16 .. 65536 rows, 64 .. 2048 columns and 16 .. 131072 k at every shape and cut (one plane; three: 75): the pick is 4 % (1 %)
// slower than the best one on average and 28 % at worst.
struct Cut { int shape, splits; };
struct Cost { double fixed1, step1, fixed2, step2; };   // one workgroup on a CU, and two (0: only one fits)
Cut cut_for(int PL, int64_t M, int64_t N, int64_t nk) {
  static const Cost cost[2][3] = {{{1., .38, 1.1, .50}, {1., .72, .6, 1.06}, {2.2, 1.51, 0., 0.}}, {{2.8, .47, .9, 1.16}, {.85, 1.23, 0., 0.}, {.85, 2.26, 0., 0.}}};
  static const int cuts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
  Cut best = {0, 1};
  double least = 1e300;
  for (int c = 0; c < 3; ++c)
    for (int s : cuts) {
      if (s > 1 && nk / s < 2) break;
      const Cost& k = cost[PL == 3][c];
      const int64_t steps = (nk + s - 1) / s, used = (nk + steps - 1) / steps, n = tiles(M, N, config_bm(PL, c), config_bn(PL, c)) * used;
      const int64_t slots = k.step2 > 0. ? 512 : 256, rest = n % slots;
      const double one = k.fixed1 + steps * k.step1, two = k.fixed2 + steps * k.step2;
      const double t = (double)(n / slots) * (slots == 512 ? two : one) + (rest > 256 ? two : rest ? one : 0.) + (s > 1 ? 4. + (double)used * M * N * 4. * .4e-6 : 0.);
      if (t < least) { least = t; best = {c, s}; }
    }
  return best;
}

// where everything lies in the workspace; the same for the size query and the run
struct Plan {
  int PL, n_kstep, h_pad;                    // h_pad: features padded for a K step
  bool h_direct, w_direct;
  int64_t rows_pad;                          // tokens padded
  int64_t chunk;                             // forward: tokens per chunk
  int64_t piece, piece_pad, n_pieces;        // backward: classes
  Cut h_cut, w_cut;                          // the two products
  bool head, turned;                         // at most 64 classes; the features also transposed
  size_t off_h, off_w, off_t, off_part, off_at, off_d, off_acc, off_wacc, off_cs, off_total, bytes;
};

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

Plan make_plan(const sgpo_linear_ce_args* a, bool backward) {
  Plan q = {};
  const bool bf = a->dtype == SGPO_DTYPE_BF16;
  q.PL = bf ? 1 : 3;
  const int kstep = bf ? 64 : 32;
  q.h_pad = (int)round_up(a->H, kstep);
  q.n_kstep = q.h_pad / kstep;
  const bool whole = bf && a->H % 64 == 0;
  q.head = a->V <= 64;
  // both operands of dweight read by rows of k would be 1110 TFLOP/s, one of them 1440; a row of the transposed features is a token long,
  // and 256 of them have to lie within the 32-bit offsets of a tile's loads
  q.turned = backward && bf && !q.head && a->N <= 1 << 22;
  q.w_direct = whole && a->ld_weight % 8 == 0 && aligned16(a->weight);
  // a product that reads the features by k (dweight's) needs zeros for ignored tokens: a packed copy, unless the transposed one has them
  q.h_direct = (!backward || q.turned) && whole && a->ld_hidden % 8 == 0 && aligned16(a->hidden);
  if (q.head && !backward) q.w_direct = q.h_direct = true;
  q.rows_pad = round_up(a->N, 64);
  size_t at = 0;
  auto take = [&](size_t n) { const size_t o = at; at += (n + 255) & ~(size_t)255; return o; };
  q.off_h = take(q.h_direct ? 0 : (size_t)q.rows_pad * q.h_pad * q.PL * 2);
  q.off_w = take(q.w_direct ? 0 : (size_t)a->V * q.h_pad * q.PL * 2);
  q.off_t = take(q.turned ? (size_t)q.rows_pad * q.h_pad * 2 : 0);
  if (!backward) {
    q.off_total = take(a->reduction != SGPO_REDUCE_NONE && a->N > TOTAL_ROWS ? (size_t)((a->N + TOTAL_ROWS - 1) / TOTAL_ROWS) * sizeof(Part) : 0);
    q.bytes = at;
    if (q.head) return q;
    const int64_t tn_max = (a->V + 63) / 64;
    q.chunk = ((int64_t)1 << 24) / tn_max & ~(int64_t)255;
    if (q.chunk < 4096) q.chunk = 4096;
    if (q.chunk > a->N) q.chunk = a->N;
    auto columns = [&](int64_t n) { const int bn = config_bn(q.PL, pick(q.PL, n, a->V)); return (a->V + bn - 1) / bn; };
    size_t part = (size_t)columns(q.chunk) * q.chunk * 8;
    if (const int64_t rest = a->N % q.chunk) {   // the last, shorter chunk may take smaller tiles
      const size_t p2 = (size_t)columns(rest) * rest * 8;
      if (p2 > part) part = p2;
    }
    q.off_part = take(part);
    q.off_at = take((size_t)q.chunk * 4);
  } else {
    int64_t piece = ((int64_t)1 << 27) / q.rows_pad & ~(int64_t)255;
    if (piece < 1024) piece = 1024;
    if (piece > a->V) piece = a->V;
    q.piece = piece;
    q.piece_pad = round_up(piece, 64);
    q.n_pieces = (a->V + piece - 1) / piece;
    q.off_d = take((size_t)q.rows_pad * q.piece_pad * q.PL * 2);
    q.h_cut = cut_for(q.PL, a->N, a->H, q.piece_pad / kstep);
    q.w_cut = cut_for(q.PL, piece, a->H, q.rows_pad / kstep);
    q.off_acc = take(q.h_cut.splits > 1 || q.n_pieces > 1 ? (size_t)q.h_cut.splits * a->N * round_up(a->H, 4) * 4 : 0);
    q.off_wacc = take(q.w_cut.splits > 1 ? (size_t)q.w_cut.splits * piece * round_up(a->H, 4) * 4 : 0);
    int bm = config_bm(q.PL, pick(q.PL, a->N, piece));
    if (a->V % piece) { const int b2 = config_bm(q.PL, pick(q.PL, a->N, a->V % piece)); if (b2 < bm) bm = b2; }
    // a row for every workgroup of the launch: a head's runs over the padded tokens
    q.off_cs = take((size_t)(q.head ? q.rows_pad / head_rows(a->N) : (a->N + bm - 1) / bm) * piece * 4);
  }
  q.bytes = at;
  return q;
}

int check_args(const sgpo_linear_ce_args* a) {
  SGPO_REQUIRE(a, "linear_ce: null arguments");
  SGPO_REQUIRE(a->N >= 0 && a->H > 0 && a->V > 0, "linear_ce: bad sizes N=%d H=%d V=%d", a->N, a->H, a->V);
  SGPO_REQUIRE(a->N <= (1 << 30) && a->V <= (1 << 30) && a->H <= (1 << 20), "linear_ce: sizes N=%d H=%d V=%d over the supported range", a->N, a->H, a->V);
  SGPO_REQUIRE(a->dtype == SGPO_DTYPE_F32 || a->dtype == SGPO_DTYPE_BF16, "linear_ce: unknown dtype %d", a->dtype);
  SGPO_REQUIRE(a->reduction >= 0 && a->reduction <= 2, "linear_ce: unknown reduction %d", a->reduction);
  SGPO_REQUIRE(a->ld_hidden >= a->H && a->ld_weight >= a->H && a->ld_hidden < (1 << 22) && a->ld_weight < (1 << 22), "linear_ce: bad row pitch %lld / %lld for H=%d",
               (long long)a->ld_hidden, (long long)a->ld_weight, a->H);
  return SGPO_OK;
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {   // bytes; a null output overlaps nothing
  return a && b && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

int blocks_for(int64_t items) {
  const int64_t b = (items + 255) / 256;
  return (int)(b < 1 ? 1 : b > 8192 ? 8192 : b);
}

template <int PL>
int pack(const void* src, int64_t ld, int rows, int cols, bf16_t* dst, int64_t rows_out, int cols_out, const int64_t* targets, int64_t ignore, hipStream_t st) {
  const int b = blocks_for(rows_out * (cols_out / 4));
  if (PL == 3) hipLaunchKernelGGL((pack_kernel<float, PL>), dim3(b), dim3(256), 0, st, (const float*)src, ld, rows, cols, dst, rows_out, cols_out, targets, ignore);
  else hipLaunchKernelGGL((pack_kernel<bf16_t, PL>), dim3(b), dim3(256), 0, st, (const bf16_t*)src, ld, rows, cols, dst, rows_out, cols_out, targets, ignore);
  SGPO_CHECK_HIP(hipGetLastError());
  return SGPO_OK;
}

#define FOR_SHAPE(PLV, C, ...)                                         \
  switch (C) {                                                         \
    case 2: { typedef typename Shapes<PLV>::L S; __VA_ARGS__ } break;         \
    case 1: { typedef typename Shapes<PLV>::M S; __VA_ARGS__ } break;         \
    default: { typedef typename Shapes<PLV>::S S; __VA_ARGS__ } break;        \
  }

template <typename T, bool GRAD>
int head(const HeadArgs& p, hipStream_t st) {
  const int rows = head_rows(p.N);
  const bool share = rows == 16;
  const dim3 grid((unsigned)(((GRAD ? (int64_t)p.rows_pad : (int64_t)p.N) + rows - 1) / rows));
#define HEAD(NB)                                                                                                       \
  case NB:                                                                                                             \
    if (share) hipLaunchKernelGGL((head_kernel<T, NB, 4, GRAD>), grid, dim3(256), 0, st, p);                           \
    else hipLaunchKernelGGL((head_kernel<T, NB, 1, GRAD>), grid, dim3(256), 0, st, p);                                 \
    break;
  switch ((p.V + 15) / 16) { HEAD(1) HEAD(2) HEAD(3) HEAD(4) }
#undef HEAD
  SGPO_CHECK_HIP(hipGetLastError());
  return SGPO_OK;
}
HeadArgs head_args(const sgpo_linear_ce_args* a) {
  HeadArgs p = {};
  p.h = a->hidden; p.w = a->weight; p.ldh = a->ld_hidden; p.ldw = a->ld_weight; p.bias = a->bias; p.targets = a->targets; p.ignore = a->ignore_index;
  p.N = a->N; p.H = a->H; p.V = a->V;
  return p;
}

void total(const sgpo_linear_ce_args* a, const float* nll, float* loss, float* inv, char* parts, hipStream_t st) {
  if (a->reduction == SGPO_REDUCE_NONE) return;
  const int mean = a->reduction == SGPO_REDUCE_MEAN;
  if (a->N <= TOTAL_ROWS) {
    hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, st, nll, a->targets, a->ignore_index, a->N, mean, loss, inv);
    return;
  }
  const int n = (a->N + TOTAL_ROWS - 1) / TOTAL_ROWS;
  hipLaunchKernelGGL(parts_kernel, dim3(n), dim3(1024), 0, st, nll, a->targets, a->ignore_index, a->N, (Part*)parts);
  hipLaunchKernelGGL(join_total_kernel, dim3(1), dim3(1024), 0, st, (const Part*)parts, n, mean, loss, inv);
}

template <int PL>
int forward(const sgpo_linear_ce_args* a, const Plan& q, float* nll, float* lse, float* loss, float* inv, char* ws, hipStream_t st) {
  if (q.head) {
    HeadArgs p = head_args(a);
    p.nll = nll; p.lse = lse;
    const int rc = PL == 1 ? head<bf16_t, false>(p, st) : head<float, false>(p, st);
    if (rc) return rc;
    total(a, nll, loss, inv, ws + q.off_total, st);
    SGPO_CHECK_HIP(hipGetLastError());
    return SGPO_OK;
  }
  tg::Operand h{(const bf16_t*)a->hidden, a->ld_hidden, a->N, 0}, w{(const bf16_t*)a->weight, a->ld_weight, a->V, 0};
  int rc;
  if (!q.h_direct) {
    bf16_t* d = (bf16_t*)(ws + q.off_h);
    if ((rc = pack<PL>(a->hidden, a->ld_hidden, a->N, a->H, d, a->N, q.h_pad, nullptr, 0, st))) return rc;
    h.p = d; h.ld = (int64_t)q.h_pad * PL;
  }
  if (!q.w_direct) {
    bf16_t* d = (bf16_t*)(ws + q.off_w);
    if ((rc = pack<PL>(a->weight, a->ld_weight, a->V, a->H, d, a->V, q.h_pad, nullptr, 0, st))) return rc;
    w.p = d; w.ld = (int64_t)q.h_pad * PL;
  }
  float2* part = (float2*)(ws + q.off_part);
  float* at = (float*)(ws + q.off_at);
  for (int64_t r0 = 0; r0 < a->N; r0 += q.chunk) {
    const int n = (int)(a->N - r0 < q.chunk ? a->N - r0 : q.chunk);
    LossArgs p{{h.p + r0 * h.ld, h.ld, n, 0}, w, a->bias, a->targets, a->ignore_index, (int)r0, n, 0, a->V, q.n_kstep};
    int tn = 0;
    FOR_SHAPE(PL, pick(PL, n, a->V), {
      const int tm = (n + S::BM - 1) / S::BM;
      tn = (a->V + S::BN - 1) / S::BN;
      ALLOW((lse_kernel<S>), S::LDS);
      hipLaunchKernelGGL((lse_kernel<S>), dim3((unsigned)tm * tn), dim3(S::THREADS), S::LDS, st, p, tm, tn, part, at);
    })
    hipLaunchKernelGGL(finish_kernel, dim3((n + 15) / 16), dim3(256), 0, st, part, n, tn, at, a->targets + r0, a->ignore_index, a->V, nll + r0, lse + r0);
  }
  total(a, nll, loss, inv, ws + q.off_total, st);
  SGPO_CHECK_HIP(hipGetLastError());
  return SGPO_OK;
}

template <int PL, int KA, int KB>
int product(MmArgs p, int shape, int splits, hipStream_t st) {
  p.nk_split = (p.nk + splits - 1) / splits;
  const int used = (p.nk + p.nk_split - 1) / p.nk_split;
#define PRODUCT(K)                                                                                                                            \
  {                                                                                                                                           \
    typedef typename Shapes<PL>::K S;                                                                                                         \
    const int tm = (p.M + S::BM - 1) / S::BM, tn = (p.N + S::BN - 1) / S::BN;                                                                 \
    ALLOW((mm_kernel<S, KA, KB>), S::LDS);                                                                                                    \
    hipLaunchKernelGGL((mm_kernel<S, KA, KB>), dim3((unsigned)tm * tn, used), dim3(S::WG_THREADS), S::LDS, st, p, tm, tn);                    \
  }
  if (shape == 2) PRODUCT(L) else if (shape == 1) PRODUCT(M) else PRODUCT(P)
#undef PRODUCT
  SGPO_CHECK_HIP(hipGetLastError());
  return used;
}

struct Sums {
  SumJobs jobs = {};
  int n = 0;
  void add(const float* src, int64_t slab, int n_slabs, int64_t rows, int cols, int64_t ld, void* out, int out_bf16, Factor factor = Factor{nullptr, nullptr}) {
    const int64_t total = rows * cols;
    const int spread = total >= 65536 || n_slabs <= 16 ? 1 : n_slabs <= 128 ? 8 : 32;
    const int64_t blocks = (total * spread + 255) / 256;
    jobs.j[n++] = SumJob{src, out, slab, ld, total, n_slabs, cols, out_bf16, spread, (int)(blocks < 8192 ? blocks : 8192), factor};
  }
  void run(hipStream_t st) {
    int blocks = 0;
    for (int i = 0; i < n; ++i) blocks += jobs.j[i].blocks;
    if (blocks) hipLaunchKernelGGL(sum_kernel, dim3(blocks), dim3(256), 0, st, jobs);
    *this = Sums();
  }
};

template <int PL>
int backward(const sgpo_linear_ce_args* a, const Plan& q, const float* lse, const float* g, const float* inv, void* dh, void* dw, float* db, char* ws, hipStream_t st) {
  const bool bf = PL == 1;
  const int kstep = bf ? 64 : 32, esz = bf ? 2 : 4;
  int rc;
  bf16_t *hp = (bf16_t*)(ws + q.off_h), *ht = (bf16_t*)(ws + q.off_t), *d = (bf16_t*)(ws + q.off_d);
  tg::Operand h{(const bf16_t*)a->hidden, a->ld_hidden, a->N, 0}, w{(const bf16_t*)a->weight, a->ld_weight, a->V, 0};
  if (!q.h_direct) {
    if (!q.head && (rc = pack<PL>(a->hidden, a->ld_hidden, a->N, a->H, hp, q.rows_pad, q.h_pad, a->targets, a->ignore_index, st))) return rc;
    h.p = hp; h.ld = (int64_t)q.h_pad * PL;
  }
  if (q.turned && dw) {
    SGPO_REQUIRE(q.h_pad / 64 <= 65535, "linear_ce_backward: H=%d", a->H);
    hipLaunchKernelGGL(transpose_kernel, dim3((unsigned)(q.rows_pad / 64), q.h_pad / 64), dim3(256), 0, st, (const bf16_t*)a->hidden, a->ld_hidden, a->N, a->H, ht, q.rows_pad,
                       a->targets, a->ignore_index);
  }
  if (!q.w_direct && (dh || !q.head)) {
    bf16_t* p = (bf16_t*)(ws + q.off_w);
    if ((rc = pack<PL>(a->weight, a->ld_weight, a->V, a->H, p, a->V, q.h_pad, nullptr, 0, st))) return rc;
    w.p = p; w.ld = (int64_t)q.h_pad * PL;
  }
  float *acc = (float*)(ws + q.off_acc), *wacc = (float*)(ws + q.off_wacc), *cs = (float*)(ws + q.off_cs);
  const int64_t ldf = round_up(a->H, 4);
  const bool via = q.h_cut.splits > 1 || q.n_pieces > 1;
  int h_used = 1;
  Sums sums;
  const Factor factor = a->reduction == SGPO_REDUCE_NONE ? Factor{nullptr, nullptr} : Factor{g, inv};
  for (int64_t v0 = 0; v0 < a->V; v0 += q.piece) {
    const int nc = (int)(a->V - v0 < q.piece ? a->V - v0 : q.piece);
    const int nc_pad = (int)round_up(nc, 64);
    int parts = 0;
    if (q.head) {
      HeadArgs p = head_args(a);
      p.lse = const_cast<float*>(lse); p.g = g; p.g_rows = a->reduction == SGPO_REDUCE_NONE;
      p.rows_pad = (int)q.rows_pad; p.h_pad = q.h_pad; p.d = d; p.hp = dw ? hp : nullptr; p.col_sums = db ? cs : nullptr;
      if ((rc = PL == 1 ? head<bf16_t, true>(p, st) : head<float, true>(p, st))) return rc;
      parts = (a->N + head_rows(a->N) - 1) / head_rows(a->N);   // further rows, of padding, hold zeros
    } else {
      LossArgs p{h, {w.p + v0 * w.ld, w.ld, (int)(a->V - v0), 0}, a->bias, a->targets, a->ignore_index, 0, a->N, (int)v0, nc, q.n_kstep};
      FOR_SHAPE(PL, pick(PL, a->N, nc), {
        parts = (a->N + S::BM - 1) / S::BM;
        const int tn = (nc + S::BN - 1) / S::BN;
        ALLOW((grad_kernel<S>), S::LDS);
        hipLaunchKernelGGL((grad_kernel<S>), dim3((unsigned)parts * tn), dim3(S::THREADS), S::LDS, st, p, parts, tn, lse, g, a->reduction == SGPO_REDUCE_NONE, d,
                           (int)q.rows_pad, nc_pad, db ? cs : nullptr);
      })
    }
    if (db) sums.add(cs, nc, parts, 1, nc, nc, db + v0, 0, factor);
    if (dh) {
      // the first piece decides how many slabs there are; later ones add to them
      MmArgs m{{d, (int64_t)nc_pad * PL, a->N, 0}, {w.p + v0 * w.ld, w.ld, nc, q.h_pad * PL}, a->N, a->H, nc_pad / kstep, 0,
               via ? (void*)acc : dh, via ? ldf : a->H, via ? (int64_t)a->N * ldf : 0, factor, a->targets, a->ignore_index, !via && bf, v0 > 0};
      const int used = product<PL, tg::KC, tg::KM>(m, q.h_cut.shape, v0 == 0 ? q.h_cut.splits : h_used, st);
      if (used < 0) return used;
      if (v0 == 0) h_used = used;
      if (via && v0 + nc == a->V) sums.add(acc, (int64_t)a->N * ldf, h_used, a->N, a->H, ldf, dh, bf);
    }
    if (dw) {
      const bool slabs = q.w_cut.splits > 1;
      void* out = (char*)dw + v0 * a->H * esz;
      MmArgs m{{d, (int64_t)nc_pad * PL, (int)q.rows_pad, nc_pad * PL}, {hp, (int64_t)q.h_pad * PL, (int)q.rows_pad, q.h_pad * PL}, nc, a->H, (int)(q.rows_pad / kstep), 0,
               slabs ? (void*)wacc : out, slabs ? ldf : a->H, slabs ? (int64_t)nc * ldf : 0, factor, nullptr, 0, !slabs && bf, 0};
      if (q.turned) m.b = tg::Operand{ht, q.rows_pad, q.h_pad, 0};
      const int used = q.turned ? product<PL, tg::KM, tg::KC>(m, q.w_cut.shape, q.w_cut.splits, st) : product<PL, tg::KM, tg::KM>(m, q.w_cut.shape, q.w_cut.splits, st);
      if (used < 0) return used;
      if (slabs) sums.add(wacc, (int64_t)nc * ldf, used, nc, a->H, ldf, out, bf);
    }
    sums.run(st);
  }
  SGPO_CHECK_HIP(hipGetLastError());
  return SGPO_OK;
}

}  // namespace

extern "C" size_t sgpo_linear_ce_workspace_bytes(const sgpo_linear_ce_args* a, int backward) {
  if (check_args(a) || a->N == 0) return 0;
  return make_plan(a, backward != 0).bytes;
}

extern "C" int sgpo_linear_ce_forward(const sgpo_linear_ce_args* a, float* nll, float* lse, float* loss, float* inv_count, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  int rc = check_args(a);
  if (rc) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  SGPO_REQUIRE(a->reduction == SGPO_REDUCE_NONE || (loss && inv_count), "linear_ce_forward: null loss / inv_count");
  if (a->N == 0) {   // no token: no loss
    total(a, nll, loss, inv_count, nullptr, st);
    SGPO_CHECK_HIP(hipGetLastError());
    return SGPO_OK;
  }
  SGPO_REQUIRE(a->hidden && a->weight && a->targets && nll && lse, "linear_ce_forward: null argument");
  const Plan q = make_plan(a, false);
  SGPO_REQUIRE((uintptr_t)workspace % 256 == 0, "linear_ce_forward: the workspace must be 256-byte aligned");
  if (q.bytes && (!workspace || workspace_bytes < q.bytes)) { sgpo_set_error("linear_ce_forward: workspace %zu < %zu", workspace_bytes, q.bytes); return SGPO_ERR_WORKSPACE; }
  return q.PL == 1 ? forward<1>(a, q, nll, lse, loss, inv_count, (char*)workspace, st) : forward<3>(a, q, nll, lse, loss, inv_count, (char*)workspace, st);
}

extern "C" int sgpo_linear_ce_backward(const sgpo_linear_ce_args* a, const float* lse, const float* grad_out, const float* inv_count, void* dhidden,
                                       void* dweight, float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_args(a);
  if (rc) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (a->N == 0) {   // no token: no gradient
    const int64_t words = (int64_t)a->V * a->H * (a->dtype == SGPO_DTYPE_BF16 ? 2 : 4) / 4, odd = (int64_t)a->V * a->H % 2;
    if (dweight) {
      if (words) hipLaunchKernelGGL(fill_kernel, dim3(blocks_for(words)), dim3(256), 0, st, (float*)dweight, words, 0.f);
      if (a->dtype == SGPO_DTYPE_BF16 && odd)
        { Sums one; one.add(nullptr, 0, 0, 1, 1, 1, (bf16_t*)dweight + words * 2, 1); one.run(st); }
    }
    if (dbias) hipLaunchKernelGGL(fill_kernel, dim3(blocks_for(a->V)), dim3(256), 0, st, dbias, (int64_t)a->V, 0.f);
    SGPO_CHECK_HIP(hipGetLastError());
    return SGPO_OK;
  }
  SGPO_REQUIRE(a->hidden && a->weight && a->targets && lse && grad_out && workspace, "linear_ce_backward: null argument");
  SGPO_REQUIRE(a->reduction == SGPO_REDUCE_NONE || inv_count, "linear_ce_backward: null inv_count");
  SGPO_REQUIRE((uintptr_t)workspace % 256 == 0, "linear_ce_backward: the workspace must be 256-byte aligned");
  const int64_t esz = a->dtype == SGPO_DTYPE_BF16 ? 2 : 4, hb = (int64_t)a->N * a->H * esz, wb = (int64_t)a->V * a->H * esz;
  const int64_t hin = ((a->N - 1) * a->ld_hidden + a->H) * esz, win = ((a->V - 1) * a->ld_weight + a->H) * esz;
  const struct { const void* p; int64_t n; } in[] = {{a->hidden, hin}, {a->weight, win}, {a->targets, (int64_t)a->N * 8}, {a->bias, (int64_t)a->V * 4}, {lse, (int64_t)a->N * 4},
      {grad_out, a->reduction == SGPO_REDUCE_NONE ? (int64_t)a->N * 4 : 4}, {a->reduction == SGPO_REDUCE_NONE ? nullptr : inv_count, 4}},
      out[] = {{dhidden, hb}, {dweight, wb}, {dbias, (int64_t)a->V * 4}};
  for (int o = 0; o < 3; ++o) {
    for (const auto& i : in) SGPO_REQUIRE(!overlap(out[o].p, out[o].n, i.p, i.n), "linear_ce_backward: a gradient overlaps an input");
    SGPO_REQUIRE(!overlap(out[o].p, out[o].n, out[(o + 1) % 3].p, out[(o + 1) % 3].n), "linear_ce_backward: a gradient overlaps another one");
  }
  const Plan q = make_plan(a, true);
  if (workspace_bytes < q.bytes) { sgpo_set_error("linear_ce_backward: workspace %zu < %zu", workspace_bytes, q.bytes); return SGPO_ERR_WORKSPACE; }
  const float* inv = a->reduction == SGPO_REDUCE_NONE ? nullptr : inv_count;
  return q.PL == 1 ? backward<1>(a, q, lse, grad_out, inv, dhidden, dweight, dbias, (char*)workspace, st)
                   : backward<3>(a, q, lse, grad_out, inv, dhidden, dweight, dbias, (char*)workspace, st);
}
