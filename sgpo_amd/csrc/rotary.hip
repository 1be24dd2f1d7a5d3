// Rotation of query and key heads by their positions.
//
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),   t = position * frequencies[j],  j < rot / 2
//   pair j of a head: elements (j, j + rot / 2), or (2j, 2j + 1) interleaved; elements from rot on are copied.
// The gradient is the transposed rotation (sin -> -sin).  cos and sin carry a factor `scale`.
//
// Bound by memory: every element is read and written once (q and k in one launch).  The angles of a token are formed once for
// all of its heads, in 64 bits -- at position 2^22 an fp32 product is off by a quarter radian -- reduced to one turn in 64 bits and only then
// rounded to fp32 for sin / cos.  The angle meant is the product position * frequency as 64 bits hold it, as in any 64-bit formula of the rotation: it
// is off by up to 2^-53 of itself, i.e. 2^-24 of a radian (as much as fp32's rounding of the reduced angle) at 2^29 radians and 2^-4 at 2^49.
#include <algorithm>

#include "../../include/sgpo_hip.h"
#include "common.h"

namespace {

struct FastDiv {   // n / d for n < 2^31
  uint32_t mul, shift, d;
};
FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return FastDiv{(uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s, d};
}
__device__ __forceinline__ uint32_t div_by(const FastDiv& f, uint32_t n, uint32_t& rem) {
  const uint32_t q = (uint32_t)(((uint64_t)__umulhi(n, f.mul) + n) >> f.shift);
  rem = n - q * f.d;
  return q;
}

struct Args {
  const void* in[2];       // q, k
  void* out[2];
  int64_t is[2][3], os[2][3];   // strides (elements) of batch, token, head
  const int64_t* pos;
  int64_t pos_sb, pos_sl;
  const double* freq;
  int64_t tokens;          // B * L < 2^31
  int heads_q, rot, D, per_block, units;
  float scale, sign;
  FastDiv by_units, by_heads, by_len;
};

template <typename T> __device__ __forceinline__ float up(T v);
template <> __device__ __forceinline__ float up<float>(float v) { return v; }
template <> __device__ __forceinline__ float up<bf16_t>(bf16_t v) { return bf2f(v); }
template <typename T> __device__ __forceinline__ T down(float v);
template <> __device__ __forceinline__ float down<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t down<bf16_t>(float v) { return f2bf(v); }

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

// A unit is VEC elements of a head (interleaved: VEC / 2 pairs, or copied ones) or, not interleaved and for single elements, VEC
// pairs (two runs of VEC elements, `apart` elements between them) before the units that copy.
template <typename T, int VEC, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(Args p) {
  extern __shared__ float2 table[];   // [per_block][rot / 2]
  const int half = p.rot >> 1;
  const int64_t t0 = (int64_t)blockIdx.x * p.per_block;
  const int nt = (int)(p.tokens - t0 < p.per_block ? p.tokens - t0 : p.per_block);
  for (int i = threadIdx.x; i < nt * half; i += 256) {
    const int tok = i / half, j = i - tok * half;
    uint32_t l;
    const int64_t b = div_by(p.by_len, (uint32_t)t0 + tok, l);
    const int64_t at = p.pos ? p.pos[b * p.pos_sb + l * p.pos_sl] : l;
    const double a = (double)at * p.freq[j];
    // one turn taken off in two pieces of 2 pi: the rest of the rounded product is exact to 2^-50 of a radian for any angle below 2^50
    const double n = rint(a * 0.15915494309189535);
    const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, a));
    float s, c;
    sincosf((float)r, &s, &c);
    table[i] = make_float2(c * p.scale, s * p.scale * p.sign);
  }
  __syncthreads();
  constexpr bool WHOLE = INTER && VEC > 1;   // pairs lie inside a unit
  constexpr int RUNS = WHOLE ? 1 : 2, ILP = 4;
  const int apart = INTER ? 1 : half;
  typedef Pack<T, VEC> V;
  const uint32_t total = (uint32_t)nt * p.by_heads.d * p.units;
  const int rot_units = WHOLE ? p.units : half / VEC;
  for (uint32_t base = threadIdx.x; base < total; base += 256 * ILP) {
    V x[ILP][RUNS];
    T* dst[ILP];
    uint32_t unit[ILP], tok[ILP];
#pragma unroll
    for (int k = 0; k < ILP; ++k) {
      const uint32_t i = base + k * 256;
      if (i >= total) continue;
      uint32_t head;
      const uint32_t row = div_by(p.by_units, i, unit[k]);
      tok[k] = div_by(p.by_heads, row, head);
      uint32_t l;
      const int64_t b = div_by(p.by_len, (uint32_t)t0 + tok[k], l);
      const int w = head >= (uint32_t)p.heads_q;
      const int h = w ? head - p.heads_q : head;
      const bool copied = !WHOLE && (int)unit[k] >= rot_units;
      const int e = WHOLE ? unit[k] * VEC : copied ? p.rot + (unit[k] - rot_units) * VEC : unit[k] * (INTER ? 2 : VEC);
      const T* src = reinterpret_cast<const T*>(w ? p.in[1] : p.in[0]) + b * (w ? p.is[1][0] : p.is[0][0]) + l * (w ? p.is[1][1] : p.is[0][1]) + h * (w ? p.is[1][2] : p.is[0][2]) + e;
      dst[k] = reinterpret_cast<T*>(w ? p.out[1] : p.out[0]) + b * (w ? p.os[1][0] : p.os[0][0]) + l * (w ? p.os[1][1] : p.os[0][1]) + h * (w ? p.os[1][2] : p.os[0][2]) + e;
      x[k][0] = *reinterpret_cast<const V*>(src);
      if constexpr (!WHOLE)
        if (!copied) x[k][1] = *reinterpret_cast<const V*>(src + apart);
    }
#pragma unroll
    for (int k = 0; k < ILP; ++k) {
      if (base + k * 256 >= total) continue;
      const float2* cs = table + tok[k] * half;
      if constexpr (WHOLE) {
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          const int j = (unit[k] * VEC + e) >> 1;
          if (j < half) {
            const float2 f = cs[j];
            const float a = up<T>(x[k][0].v[e]), b = up<T>(x[k][0].v[e + 1]);
            x[k][0].v[e] = down<T>(a * f.x - b * f.y);
            x[k][0].v[e + 1] = down<T>(a * f.y + b * f.x);
          }
        }
        *reinterpret_cast<V*>(dst[k]) = x[k][0];
      } else {
        if ((int)unit[k] < rot_units) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float2 f = cs[unit[k] * VEC + e];
            const float a = up<T>(x[k][0].v[e]), b = up<T>(x[k][RUNS - 1].v[e]);
            x[k][0].v[e] = down<T>(a * f.x - b * f.y);
            x[k][RUNS - 1].v[e] = down<T>(a * f.y + b * f.x);
          }
          *reinterpret_cast<V*>(dst[k] + apart) = x[k][RUNS - 1];
        }
        *reinterpret_cast<V*>(dst[k]) = x[k][0];
      }
    }
  }
}

template <typename T, int VEC, bool INTER>
int launch(Args& p, int heads, hipStream_t st) {
  const int half = p.rot / 2;
  p.units = INTER && VEC > 1 ? p.D / VEC : half / VEC + (p.D - p.rot) / VEC;
  p.by_units = fast_div(p.units);
  p.by_heads = fast_div(heads);
  // Tokens per workgroup: about two units per thread, so that a CU's workgroups overlap one's angles with another's copying (30464 tokens
  // of 16 bf16 heads of 64: 24.5 us with 8 tokens, 29.5 with 64; 41 with one, where too few units share a token's angles), but at most
  // 65536 workgroups, whose dispatch takes longer than their work (131072 tokens of 40 heads of 128: 498 us with one token, 456 with two).
  const int64_t per_token = (int64_t)heads * p.units, fit = half ? 4096 / half : 4096, fewest = (p.tokens + 65535) / 65536;
  int64_t t = (512 + per_token - 1) / per_token;
  if (t < fewest) t = fewest;
  if (t > fit) t = fit;
  if (t < 1) t = 1;
  p.per_block = (int)t;
  const int64_t grid = (p.tokens + t - 1) / t;
  SGPO_REQUIRE(grid < 0x7fffffff && (int64_t)heads * p.units * t < 0x7fffffff, "rotary: too many tokens or heads");
  hipLaunchKernelGGL((rotary_kernel<T, VEC, INTER>), dim3((unsigned)grid), dim3(256), (size_t)t * half * sizeof(float2), st, p);
  SGPO_CHECK_HIP(hipGetLastError());
  return SGPO_OK;
}

template <typename T>
int run(const sgpo_rotary_args* a, hipStream_t st) {
  Args p = {};
  p.pos = a->positions; p.pos_sb = a->pos_stride_b; p.pos_sl = a->pos_stride_l;
  p.freq = a->frequencies;
  p.tokens = (int64_t)a->B * a->L;
  p.by_len = fast_div(a->L);
  p.heads_q = a->heads_q; p.rot = a->rot; p.D = a->head_dim;
  p.scale = a->scale; p.sign = a->inverse ? -1.f : 1.f;
  // the widest run that divides every offset: base pointers, strides and, not interleaved, the half distance
  const int most = 16 / sizeof(T);
  uint64_t off = a->head_dim;
  if (!a->interleaved) off |= a->rot / 2 | a->rot;
  const int heads[2] = {a->heads_q, a->heads_k};
  for (int w = 0; w < 2; ++w) {
    p.in[w] = w ? a->k : a->q; p.out[w] = w ? a->k_out : a->q_out;
    for (int i = 0; i < 3; ++i) {
      p.is[w][i] = w ? a->k_stride[i] : a->q_stride[i];
      p.os[w][i] = w ? a->k_out_stride[i] : a->q_out_stride[i];
      const int dim = i == 0 ? a->B : i == 1 ? a->L : heads[w];
      if (heads[w] && dim > 1) off |= (uint64_t)p.is[w][i] | (uint64_t)p.os[w][i];
    }
    if (heads[w]) off |= (uintptr_t)p.in[w] / sizeof(T) | (uintptr_t)p.out[w] / sizeof(T);
  }
  int vec = most;
  while (vec > 1 && off % vec) vec >>= 1;
  const int h = heads[0] + heads[1];
  if (a->interleaved) {
    if (vec == 8) { if constexpr (sizeof(T) == 2) return launch<T, 8, true>(p, h, st); }
    if (vec >= 4) return launch<T, 4, true>(p, h, st);
    if (vec >= 2) return launch<T, 2, true>(p, h, st);
    return launch<T, 1, true>(p, h, st);
  }
  if (vec == 8) { if constexpr (sizeof(T) == 2) return launch<T, 8, false>(p, h, st); }
  if (vec >= 4) return launch<T, 4, false>(p, h, st);
  if (vec >= 2) return launch<T, 2, false>(p, h, st);
  return launch<T, 1, false>(p, h, st);
}

// Heads in memory: four dimensions, the last one contiguous.  Host side of the in-place call: what a workgroup writes must be nothing that
// another one reads.
struct View {
  uintptr_t at;
  int64_t n[4], s[4];   // elements; a dimension of one element has no stride
  int64_t extent() const {
    int64_t e = 1;
    for (int i = 0; i < 4; ++i) e += (n[i] - 1) * (s[i] < 0 ? -s[i] : s[i]);
    return e;
  }
};
View view_of(const void* p, const int64_t* stride, int B, int L, int heads, int D) {
  return View{(uintptr_t)p, {B, L, heads, D}, {stride[0], stride[1], stride[2], 1}};
}
// is r = sum of delta_i * s_i with -(nb_i - 1) <= delta_i <= na_i - 1, over the dimensions from i on (strides descending)?
bool reachable(int64_t r, const int64_t (&s)[4], const int64_t (&na)[4], const int64_t (&nb)[4], int i) {
  if (i == 4) return r == 0;
  int64_t up = 0, down = 0;   // what the dimensions behind this one can add
  for (int j = i + 1; j < 4; ++j) { up += (na[j] - 1) * s[j]; down += (nb[j] - 1) * s[j]; }
  if (s[i] == 0) return reachable(r, s, na, nb, i + 1);
  auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  int64_t lo = -floor_div(up - r, s[i]), hi = floor_div(r + down, s[i]);   // r - delta s within [-down, up]
  if (lo < -(nb[i] - 1)) lo = -(nb[i] - 1);
  if (hi > na[i] - 1) hi = na[i] - 1;
  for (int64_t d = lo; d <= hi; ++d)
    if (reachable(r - d * s[i], s, na, nb, i + 1)) return true;
  return false;
}
// no two elements at one place: each stride reaches over all that the smaller ones span
bool apart(const View& v) {
  int order[4] = {0, 1, 2, 3};
  std::sort(order, order + 4, [&](int a, int b) { return v.s[a] < v.s[b]; });
  int64_t span = 1;
  for (int i : order) {
    if (v.n[i] <= 1) continue;
    if (v.s[i] < span) return false;
    span += (v.n[i] - 1) * v.s[i];
  }
  return true;
}
// may a and b share memory?  Exact for views of one packed tensor (the same strides); any others whose address ranges meet count as sharing.
bool share(const View& a, const View& b, size_t esz) {
  for (int i = 0; i < 3; ++i) if (a.s[i] < 0 || b.s[i] < 0) return true;
  if (a.at + a.extent() * esz <= b.at || b.at + b.extent() * esz <= a.at) return false;
  const int64_t bytes = (int64_t)(a.at - b.at);
  if (bytes % (int64_t)esz) return true;
  int order[4] = {0, 1, 2, 3};
  int64_t s[4];
  for (int i = 0; i < 4; ++i) {
    if (a.n[i] > 1 && b.n[i] > 1 && a.s[i] != b.s[i]) return true;
    s[i] = a.n[i] > 1 ? a.s[i] : b.n[i] > 1 ? b.s[i] : 0;
  }
  std::sort(order, order + 4, [&](int x, int y) { return s[x] > s[y]; });
  int64_t so[4], na[4], nb[4];
  for (int i = 0; i < 4; ++i) { so[i] = s[order[i]]; na[i] = a.n[order[i]]; nb[i] = b.n[order[i]]; }
  return reachable(-bytes / (int64_t)esz, so, na, nb, 0);   // a.at + delta s = b.at
}

int check_memory(const sgpo_rotary_args* a) {
  const size_t esz = a->dtype == SGPO_DTYPE_BF16 ? 2 : 4;
  View in[2], out[2];
  const int heads[2] = {a->heads_q, a->heads_k};
  for (int w = 0; w < 2; ++w) {
    if (!heads[w]) continue;
    in[w] = view_of(w ? a->k : a->q, w ? a->k_stride : a->q_stride, a->B, a->L, heads[w], a->head_dim);
    out[w] = view_of(w ? a->k_out : a->q_out, w ? a->k_out_stride : a->q_out_stride, a->B, a->L, heads[w], a->head_dim);
    SGPO_REQUIRE(in[w].at && out[w].at && in[w].at % esz == 0 && out[w].at % esz == 0, "rotary: null or misaligned heads");
    SGPO_REQUIRE(apart(out[w]), "rotary: elements of the output overlap");
  }
  for (int w = 0; w < 2; ++w)
    for (int u = 0; u < 2; ++u) {
      if (!heads[w] || !heads[u]) continue;
      bool same = w == u && in[u].at == out[w].at;
      for (int i = 0; i < 3; ++i) same = same && (in[u].n[i] <= 1 || in[u].s[i] == out[w].s[i]);
      SGPO_REQUIRE(same || !share(out[w], in[u], esz), "rotary: an output overlaps %s", w == u ? "its input without being it" : "the other input");
    }
  SGPO_REQUIRE(!heads[0] || !heads[1] || !share(out[0], out[1], esz), "rotary: q_out and k_out overlap");
  return SGPO_OK;
}

}  // namespace

extern "C" int sgpo_rotary(const sgpo_rotary_args* a, void* stream) {
  SGPO_REQUIRE(a, "rotary: null arguments");
  SGPO_REQUIRE(a->B >= 0 && a->L >= 0 && a->heads_q >= 0 && a->heads_k >= 0, "rotary: negative size");
  SGPO_REQUIRE(a->head_dim >= 1 && a->head_dim <= 4096 && a->rot >= 0 && a->rot % 2 == 0 && a->rot <= a->head_dim, "rotary: rot=%d must be even and at most head_dim=%d (1..4096)",
               a->rot, a->head_dim);
  SGPO_REQUIRE(a->dtype == SGPO_DTYPE_F32 || a->dtype == SGPO_DTYPE_BF16, "rotary: unknown dtype %d", a->dtype);
  const int64_t heads = (int64_t)a->heads_q + a->heads_k;
  if ((int64_t)a->B * a->L == 0 || heads == 0) return SGPO_OK;
  SGPO_REQUIRE(heads < 0x7fffffff, "rotary: %lld heads in one call", (long long)heads);
  SGPO_REQUIRE((int64_t)a->B * a->L < 0x7fffffff, "rotary: B * L = %lld tokens in one call", (long long)a->B * a->L);
  if (const int rc = check_memory(a)) return rc;
  SGPO_REQUIRE(a->rot == 0 || a->frequencies, "rotary: null frequencies");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return a->dtype == SGPO_DTYPE_BF16 ? run<bf16_t>(a, st) : run<float>(a, st);
}
