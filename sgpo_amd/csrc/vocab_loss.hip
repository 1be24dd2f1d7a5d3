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
// 2 N V H operations forward and 6 backward; everything but the operands and gradients stays in caches or registers.
//
// bf16 operands: one plane; d is rounded to bf16 once (relative error 2^-8 at most per term, of the size of the outputs' own
// rounding), sums in fp32.  fp32 operands: three planes, i.e. products and d with 24 bits.
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
#pragma unroll
  for (int y = 0; y < S::NT; ++y)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = n0 + (wn * S::NT + y) * 16 + 4 * l4 + q;
      const bool in = n < p.n_cls;
      const float b = in && p.bias ? p.bias[p.v0 + n] : 0.f;
#pragma unroll
      for (int x = 0; x < S::MT; ++x) acc[x][y][q] = in ? acc[x][y][q] + b : -INFINITY;
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
      const int64_t t = p.targets[p.r0 + m] - p.v0 - n0;
      if (t >= 0 && t < S::BN && p.targets[p.r0 + m] != p.ignore) {
#pragma unroll
        for (int y = 0; y < S::NT; ++y)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if ((wn * S::NT + y) * 16 + 4 * l4 + q == (int)t && n0 + (int)t < p.n_cls) at_target[m] = acc[x][y][q];
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

// joins a token's pairs: 64 tokens per workgroup, four waves share a token's tile columns
__global__ __launch_bounds__(256) void finish_kernel(const float2* part, int n_rows, int tn, const float* at_target, const int64_t* targets,
                                                     int64_t ignore, int V, float* nll, float* lse) {
  __shared__ float2 share[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int m = blockIdx.x * 64 + lane;
  float a = -INFINITY, s = 0.f;
  if (m < n_rows)
    for (int i = w; i < tn; i += 4) {
      const float2 b = part[(int64_t)i * n_rows + m];
      join(a, s, b.x, b.y);
    }
  share[w][lane] = make_float2(a, s);
  __syncthreads();
  if (w == 0 && m < n_rows) {
#pragma unroll
    for (int i = 1; i < 4; ++i) join(a, s, share[i][lane].x, share[i][lane].y);
    const float l = a + logf(s);
    const int64_t t = targets[m];
    lse[m] = l;
    // a target that is no class has no loss: NaN, so that the step shows it
    nll[m] = t == ignore ? 0.f : (t < 0 || t >= V) ? __builtin_nanf("") : l - at_target[m];
  }
}

// loss[0] = sum of nll (reduction 2) or its mean over the tokens with a loss (1; 0 if there are none); inv[0] = the factor on every token's gradient
__global__ __launch_bounds__(1024) void total_kernel(const float* nll, const int64_t* targets, int64_t ignore, int N, int mean, float* loss, float* inv) {
  __shared__ double ssum[16];
  __shared__ int scnt[16];
  double s = 0.0;
  int c = 0;
  for (int i = threadIdx.x; i < N; i += 1024) {
    s += (double)nll[i];
    c += targets[i] != ignore;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { s += __shfl_xor(s, o); c += __shfl_xor(c, o); }
  if ((threadIdx.x & 63) == 0) { ssum[threadIdx.x >> 6] = s; scnt[threadIdx.x >> 6] = c; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) { s += ssum[i]; c += scnt[i]; }
    const int n = mean ? (c > 0 ? c : 1) : 1;
    loss[0] = (float)(s / n);
    inv[0] = 1.f / (float)n;
  }
}

// ----------------------------------------------------------------------------------------------------------- backward
// d of a piece of the vocabulary into d [rows_pad][cols_pad] planes (zero beyond the tokens and classes); column sums per row tile
template <class S>
__global__ __launch_bounds__(S::THREADS, 2) void grad_kernel(LossArgs p, int tm, int tn, const float* lse, const float* g,
                                                               int g_rows, const float* inv, bf16_t* d, int rows_pad, int cols_pad,
                                                               float* col_sums) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int im, in;
  tg::tile_of(blockIdx.x, tm, tn, im, in);
  const int m0 = im * S::BM, n0 = in * S::BN;
  f32x4 acc[S::MT][S::NT];
  logits<S>(p, m0, n0, smem, acc);
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = (int)threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  const float f = inv ? inv[0] : 1.f;
  float cs[S::NT][4];
#pragma unroll
  for (int y = 0; y < S::NT; ++y)
#pragma unroll
    for (int q = 0; q < 4; ++q) cs[y][q] = 0.f;
#pragma unroll
  for (int x = 0; x < S::MT; ++x) {
    const int m = m0 + (wm * S::MT + x) * 16 + l16;
    const bool in_rows = m < p.n_rows;
    const int64_t t = in_rows ? p.targets[m] : p.ignore;
    const bool keep = in_rows && t != p.ignore;
    const bool bad = keep && (t < 0 || t >= (int64_t)p.w.rows + p.v0);
    const float l = keep ? lse[m] : 0.f;
    const float gm = keep ? (bad ? __builtin_nanf("") : g[g_rows ? m : 0] * f) : 0.f;
    const int tl = (int)(keep ? (t - p.v0 < 0 || t - p.v0 > 0x7fffffff ? -1 : t - p.v0) : -1);
#pragma unroll
    for (int y = 0; y < S::NT; ++y) {
      const int n = n0 + (wn * S::NT + y) * 16 + 4 * l4;
      float v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float e = __builtin_amdgcn_exp2f((acc[x][y][q] - l) * LOG2E);
        v[q] = keep && n + q < p.n_cls ? gm * (e - (n + q == tl ? 1.f : 0.f)) : 0.f;
        cs[y][q] += v[q];
      }
      if (m < rows_pad && n < cols_pad) tg::store4<S::PL>(d + (int64_t)m * cols_pad * S::PL, n, v);
    }
  }
  if (!col_sums) return;
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

// C tile of a product, K split over gridDim.y slabs: fp32 (added to what is there if `add`) or rounded to bf16
struct MmArgs {
  tg::Operand a, b;
  int M, N, nk, nk_split;
  void* out;
  int64_t ldo, slab;
  int out_bf16, add, vec;   // vec: rows start 16-B (fp32) / 8-B (bf16) aligned
};

template <class S, int KA, int KB>
__global__ __launch_bounds__(S::THREADS, 2) void mm_kernel(MmArgs p, int tm, int tn) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int im, in;
  tg::tile_of(blockIdx.x, tm, tn, im, in);
  const int m0 = im * S::BM, n0 = in * S::BN;
  const int k0 = blockIdx.y * p.nk_split, nk = min(p.nk_split, p.nk - k0);
  f32x4 acc[S::MT][S::NT];
  tg::clear<S>(acc);
  tg::run<S, KA, KB>(p.a, p.b, m0, n0, k0, nk, smem, acc);
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = (int)threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
  for (int x = 0; x < S::MT; ++x) {
    const int m = m0 + (wm * S::MT + x) * 16 + l16;
    if (m >= p.M) continue;
#pragma unroll
    for (int y = 0; y < S::NT; ++y) {
      const int n = n0 + (wn * S::NT + y) * 16 + 4 * l4;
      f32x4 v = acc[x][y];
      if (p.out_bf16) {
        bf16_t* o = reinterpret_cast<bf16_t*>(p.out) + m * p.ldo + n;
        if (p.vec && n + 4 <= p.N) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        else
#pragma unroll
          for (int q = 0; q < 4; ++q) if (n + q < p.N) o[q] = f2bf(v[q]);
      } else {
        float* o = reinterpret_cast<float*>(p.out) + blockIdx.y * p.slab + m * p.ldo + n;
        if (p.vec && n + 4 <= p.N) {
          if (p.add) v += *reinterpret_cast<const f32x4*>(o);
          *reinterpret_cast<f32x4*>(o) = v;
        } else
#pragma unroll
          for (int q = 0; q < 4; ++q) if (n + q < p.N) o[q] = p.add ? o[q] + v[q] : v[q];
      }
    }
  }
}

// out[r][c] = sum over slabs of src[s][r][c]; src rows have ld elements
__global__ __launch_bounds__(256) void sum_kernel(const float* src, int64_t slab, int n_slabs, int rows, int cols, int64_t ld, void* out, int out_bf16) {
  const int64_t total = (int64_t)rows * cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / cols, c = i - r * cols;
    float s = 0.f;
    for (int k = 0; k < n_slabs; ++k) s += src[k * slab + r * ld + c];
    if (out_bf16) reinterpret_cast<bf16_t*>(out)[i] = f2bf(s);
    else reinterpret_cast<float*>(out)[i] = s;
  }
}

__global__ __launch_bounds__(256) void fill_kernel(float* p, int64_t n, float v) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = v;
}

// ---------------------------------------------------------------------------------------------------------- host side
template <int PL> struct Shapes;
template <> struct Shapes<1> {
  typedef tg::Shape<256, 256, 2, 4, 1, 2> L;
  typedef tg::Shape<128, 128, 2, 2, 1, 2> M;
  typedef tg::Shape<64, 64, 2, 2, 1, 4> S;
};
template <> struct Shapes<3> {
  typedef tg::Shape<256, 128, 4, 2, 3, 2> L;
  typedef tg::Shape<128, 128, 2, 4, 3, 2> M;
  typedef tg::Shape<64, 64, 2, 2, 3, 2> S;
};

inline int64_t tiles(int64_t m, int64_t n, int bm, int bn) { return (m + bm - 1) / bm * ((n + bn - 1) / bn); }

// the largest tile that still gives most of the CUs one
template <int PL>
int pick(int64_t M, int64_t N) {
  if (tiles(M, N, Shapes<PL>::L::BM, Shapes<PL>::L::BN) >= 160) return 2;
  return tiles(M, N, Shapes<PL>::M::BM, Shapes<PL>::M::BN) >= 160 ? 1 : 0;
}

template <typename K>
int allow_lds(K kernel, int bytes) {
  SGPO_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return SGPO_OK;
}

// where everything lies in the workspace; the same for the size query and the run
struct Plan {
  int PL, n_kstep, h_pad;                    // h_pad: features padded for a K step
  bool h_direct, w_direct;
  int64_t rows_pad;                          // tokens padded
  int64_t chunk, tn;                         // forward: tokens per chunk, tile columns
  int64_t piece, piece_pad, n_pieces;        // backward: classes
  int h_splits, w_splits;                    // K splits of the two products
  size_t off_h, off_w, off_part, off_at, off_d, off_acc, off_wacc, off_cs, bytes;
};

int config_bn(int PL, int c) { return PL == 1 ? (c == 2 ? 256 : c == 1 ? 128 : 64) : (c ? 128 : 64); }
int config_bm(int PL, int c) { return c == 2 ? 256 : c == 1 ? 128 : 64; }
int pick_pl(int PL, int64_t M, int64_t N) { return PL == 1 ? pick<1>(M, N) : pick<3>(M, N); }

// enough slabs of K to give every CU work, at least four steps each
int splits_for(int PL, int64_t M, int64_t N, int64_t nk) {
  const int c = pick_pl(PL, M, N);
  const int64_t t = tiles(M, N, config_bm(PL, c), config_bn(PL, c));
  int64_t s = 384 / t;
  if (s > nk / 4) s = nk / 4;
  if (s > 64) s = 64;
  return s < 1 ? 1 : (int)s;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

Plan make_plan(const sgpo_linear_ce_args* a, bool backward) {
  Plan q = {};
  const bool bf = a->dtype == SGPO_DTYPE_BF16;
  q.PL = bf ? 1 : 3;
  const int kstep = bf ? 64 : 32;
  q.h_pad = (int)round_up(a->H, 64);
  q.n_kstep = q.h_pad / kstep;
  const bool whole = bf && a->H % 64 == 0;
  q.w_direct = whole && a->ld_weight % 8 == 0 && aligned16(a->weight);
  q.h_direct = !backward && whole && a->ld_hidden % 8 == 0 && aligned16(a->hidden);
  q.rows_pad = round_up(a->N, 64);
  size_t at = 0;
  auto take = [&](size_t n) { const size_t o = at; at += (n + 255) & ~(size_t)255; return o; };
  q.off_h = take(q.h_direct ? 0 : (size_t)q.rows_pad * q.h_pad * q.PL * 2);
  q.off_w = take(q.w_direct ? 0 : (size_t)a->V * q.h_pad * q.PL * 2);
  if (!backward) {
    const int64_t tn_max = (a->V + 63) / 64;
    q.chunk = ((int64_t)1 << 24) / tn_max & ~(int64_t)255;
    if (q.chunk < 4096) q.chunk = 4096;
    if (q.chunk > a->N) q.chunk = a->N;
    const int c = pick_pl(q.PL, q.chunk, a->V);
    q.tn = (a->V + config_bn(q.PL, c) - 1) / config_bn(q.PL, c);
    // the last, shorter chunk may take smaller tiles: room for their columns
    const int64_t rest = a->N % q.chunk;
    size_t part = (size_t)q.tn * q.chunk * 8;
    if (rest) {
      const int c2 = pick_pl(q.PL, rest, a->V);
      const size_t p2 = (size_t)((a->V + config_bn(q.PL, c2) - 1) / config_bn(q.PL, c2)) * rest * 8;
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
    q.h_splits = splits_for(q.PL, a->N, a->H, q.piece_pad / kstep);
    q.w_splits = splits_for(q.PL, piece, a->H, q.rows_pad / kstep);
    q.off_acc = take(q.h_splits > 1 || q.n_pieces > 1 ? (size_t)q.h_splits * a->N * round_up(a->H, 4) * 4 : 0);
    q.off_wacc = take(q.w_splits > 1 ? (size_t)q.w_splits * piece * round_up(a->H, 4) * 4 : 0);
    const int c = pick_pl(q.PL, a->N, piece);
    int bm = config_bm(q.PL, c);
    if (a->V % piece) { const int b2 = config_bm(q.PL, pick_pl(q.PL, a->N, a->V % piece)); if (b2 < bm) bm = b2; }
    q.off_cs = take((size_t)((a->N + bm - 1) / bm) * piece * 4);
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
#define ALLOW(kernel, bytes)                                           \
  do {                                                                 \
    static bool done = false;                                          \
    if (!done) { const int rc_ = allow_lds(kernel, bytes); if (rc_) return rc_; done = true; } \
  } while (0)

template <int PL>
int forward(const sgpo_linear_ce_args* a, const Plan& q, float* nll, float* lse, float* loss, float* inv, char* ws, hipStream_t st) {
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
    FOR_SHAPE(PL, pick<PL>(n, a->V), {
      const int tm = (n + S::BM - 1) / S::BM;
      tn = (a->V + S::BN - 1) / S::BN;
      ALLOW((lse_kernel<S>), S::LDS);
      hipLaunchKernelGGL((lse_kernel<S>), dim3((unsigned)tm * tn), dim3(S::THREADS), S::LDS, st, p, tm, tn, part, at);
    })
    hipLaunchKernelGGL(finish_kernel, dim3((n + 63) / 64), dim3(256), 0, st, part, n, tn, at, a->targets + r0, a->ignore_index, a->V, nll + r0, lse + r0);
  }
  if (a->reduction != SGPO_REDUCE_NONE)
    hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, st, nll, a->targets, a->ignore_index, a->N, a->reduction == SGPO_REDUCE_MEAN, loss, inv);
  SGPO_CHECK_HIP(hipGetLastError());
  return SGPO_OK;
}

template <int PL, int KA, int KB>
int product(MmArgs p, int splits, hipStream_t st) {
  p.nk_split = (p.nk + splits - 1) / splits;
  const int used = (p.nk + p.nk_split - 1) / p.nk_split;
  FOR_SHAPE(PL, pick<PL>(p.M, p.N), {
    const int tm = (p.M + S::BM - 1) / S::BM, tn = (p.N + S::BN - 1) / S::BN;
    ALLOW((mm_kernel<S, KA, KB>), S::LDS);
    hipLaunchKernelGGL((mm_kernel<S, KA, KB>), dim3((unsigned)tm * tn, used), dim3(S::THREADS), S::LDS, st, p, tm, tn);
  })
  SGPO_CHECK_HIP(hipGetLastError());
  return used;
}

template <int PL>
int backward(const sgpo_linear_ce_args* a, const Plan& q, const float* lse, const float* g, const float* inv, void* dh, void* dw, float* db, char* ws, hipStream_t st) {
  const bool bf = PL == 1;
  const int kstep = bf ? 64 : 32, esz = bf ? 2 : 4;
  int rc;
  bf16_t* hp = (bf16_t*)(ws + q.off_h);
  if ((rc = pack<PL>(a->hidden, a->ld_hidden, a->N, a->H, hp, q.rows_pad, q.h_pad, a->targets, a->ignore_index, st))) return rc;
  tg::Operand h{hp, (int64_t)q.h_pad * PL, a->N, 0}, w{(const bf16_t*)a->weight, a->ld_weight, a->V, 0};
  if (!q.w_direct) {
    bf16_t* d = (bf16_t*)(ws + q.off_w);
    if ((rc = pack<PL>(a->weight, a->ld_weight, a->V, a->H, d, a->V, q.h_pad, nullptr, 0, st))) return rc;
    w.p = d; w.ld = (int64_t)q.h_pad * PL;
  }
  bf16_t* d = (bf16_t*)(ws + q.off_d);
  float* acc = (float*)(ws + q.off_acc);
  float* wacc = (float*)(ws + q.off_wacc);
  float* cs = (float*)(ws + q.off_cs);
  const int64_t ldf = round_up(a->H, 4);
  const bool via = q.h_splits > 1 || q.n_pieces > 1;
  int h_used = 1;
  for (int64_t v0 = 0; v0 < a->V; v0 += q.piece) {
    const int nc = (int)(a->V - v0 < q.piece ? a->V - v0 : q.piece);
    const int nc_pad = (int)round_up(nc, 64);
    LossArgs p{h, {w.p + v0 * w.ld, w.ld, (int)(a->V - v0), 0}, a->bias, a->targets, a->ignore_index, 0, a->N, (int)v0, nc, q.n_kstep};
    int tm = 0;
    FOR_SHAPE(PL, pick<PL>(a->N, nc), {
      tm = (a->N + S::BM - 1) / S::BM;
      const int tn = (nc + S::BN - 1) / S::BN;
      ALLOW((grad_kernel<S>), S::LDS);
      hipLaunchKernelGGL((grad_kernel<S>), dim3((unsigned)tm * tn), dim3(S::THREADS), S::LDS, st, p, tm, tn, lse, g, a->reduction == SGPO_REDUCE_NONE, inv, d,
                         (int)q.rows_pad, nc_pad, db ? cs : nullptr);
    })
    if (db) hipLaunchKernelGGL(sum_kernel, dim3(blocks_for(nc)), dim3(256), 0, st, cs, (int64_t)nc, tm, 1, nc, (int64_t)nc, db + v0, 0);
    if (dh) {
      // the first piece decides how many slabs there are; later ones add to them
      MmArgs m{{d, (int64_t)nc_pad * PL, a->N, 0}, {w.p + v0 * w.ld, w.ld, nc, q.h_pad * PL}, a->N, a->H, nc_pad / kstep, 0,
               via ? (void*)acc : dh, via ? ldf : a->H, via ? (int64_t)a->N * ldf : 0, !via && bf, v0 > 0,
               via || (a->H % 4 == 0 && aligned16(dh))};
      const int used = product<PL, tg::KC, tg::KM>(m, v0 == 0 ? q.h_splits : h_used, st);
      if (used < 0) return used;
      if (v0 == 0) h_used = used;
    }
    if (dw) {
      const bool slabs = q.w_splits > 1;
      void* out = (char*)dw + v0 * a->H * esz;
      MmArgs m{{d, (int64_t)nc_pad * PL, (int)q.rows_pad, nc_pad * PL}, {hp, (int64_t)q.h_pad * PL, (int)q.rows_pad, q.h_pad * PL}, nc, a->H, (int)(q.rows_pad / kstep), 0,
               slabs ? (void*)wacc : out, slabs ? ldf : a->H, slabs ? (int64_t)nc * ldf : 0, !slabs && bf, 0,
               slabs || (a->H % 4 == 0 && aligned16(out))};
      const int used = product<PL, tg::KM, tg::KM>(m, q.w_splits, st);
      if (used < 0) return used;
      if (slabs) hipLaunchKernelGGL(sum_kernel, dim3(blocks_for((int64_t)nc * a->H)), dim3(256), 0, st, wacc, (int64_t)nc * ldf, used, nc, a->H, ldf, out, bf ? 1 : 0);
    }
  }
  if (dh && via) hipLaunchKernelGGL(sum_kernel, dim3(blocks_for((int64_t)a->N * a->H)), dim3(256), 0, st, acc, (int64_t)a->N * ldf, h_used, a->N, a->H, ldf, dh, bf ? 1 : 0);
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
    if (a->reduction != SGPO_REDUCE_NONE) hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, st, nll, a->targets, a->ignore_index, 0, a->reduction == SGPO_REDUCE_MEAN, loss, inv_count);
    SGPO_CHECK_HIP(hipGetLastError());
    return SGPO_OK;
  }
  SGPO_REQUIRE(a->hidden && a->weight && a->targets && nll && lse && workspace, "linear_ce_forward: null argument");
  const Plan q = make_plan(a, false);
  if (workspace_bytes < q.bytes) { sgpo_set_error("linear_ce_forward: workspace %zu < %zu", workspace_bytes, q.bytes); return SGPO_ERR_WORKSPACE; }
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
        hipLaunchKernelGGL(sum_kernel, dim3(1), dim3(256), 0, st, (const float*)nullptr, (int64_t)0, 0, 1, 1, (int64_t)1, (bf16_t*)dweight + words * 2, 1);
    }
    if (dbias) hipLaunchKernelGGL(fill_kernel, dim3(blocks_for(a->V)), dim3(256), 0, st, dbias, (int64_t)a->V, 0.f);
    SGPO_CHECK_HIP(hipGetLastError());
    return SGPO_OK;
  }
  SGPO_REQUIRE(a->hidden && a->weight && a->targets && lse && grad_out && workspace, "linear_ce_backward: null argument");
  SGPO_REQUIRE(a->reduction == SGPO_REDUCE_NONE || inv_count, "linear_ce_backward: null inv_count");
  const Plan q = make_plan(a, true);
  if (workspace_bytes < q.bytes) { sgpo_set_error("linear_ce_backward: workspace %zu < %zu", workspace_bytes, q.bytes); return SGPO_ERR_WORKSPACE; }
  const float* inv = a->reduction == SGPO_REDUCE_NONE ? nullptr : inv_count;
  return q.PL == 1 ? backward<1>(a, q, lse, grad_out, inv, dhidden, dweight, dbias, (char*)workspace, st)
                   : backward<3>(a, q, lse, grad_out, inv, dhidden, dweight, dbias, (char*)workspace, st);
}
