// One output tile of  C[m][n] = sum_k A[m][k] B[n][k]  on the matrix cores, for the training operators (vocab_loss.hip,
// orthogonal.hip).  Only the K loop lives here; the caller's kernel owns the accumulators and its epilogue.
//
// Numbers.  An operand is stored as PL bf16 PLANES whose sum is the value: one plane is a plain bf16 matrix, two planes leave a
// rest of at most 2^-17 |x|, three of 2^-26 |x| (an fp32 value's own half step is 2^-24).  Products of bf16 are exact in fp32.  The plane
// pairs (i, j) with i + j < PL are multiplied -- 1, 3 or 6 MFMAs per product, smallest first; the pairs left out are below 2^-16 |x y| (two planes)
// and 2^-24 |x y| (three).  The matrix cores run 16 bf16 MFMAs in the time of one fp32 MFMA of the same shape, so six bf16
// products are 2.6 times the rate of native fp32.
//
// Layouts.  The planes of a matrix are interleaved along its contiguous direction in runs of 32: element e, plane p is stored
// at (e / 32) * 32 * PL + p * 32 + e % 32.  One K step then moves the same bytes whatever PL is (64 k of one plane, 32 k of two
// or three), and one plane is the ordinary row-major layout.  An operand is read either way round:
//   KC  rows are m (or n), k contiguous: fragments by ds_read_b128, 8 consecutive k of a row per lane;
//   KM  rows are k, m (or n) contiguous: fragments by ds_read_b64_tr_b16 (the LDS transposes 4 x 16 blocks on the way to the
//       registers), so that no transposed copy of any operand ever exists in memory.
// LDS images are filled by LDS-DMA, 16 B per lane, lane-linear; bank conflicts are avoided by permuting the 16-B chunks of a
// row on the source address and again on the read.
#pragma once
#include "common.h"

namespace tg {

typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4* lds_tr_t;

enum { KC = 0, KM = 1 };

// ld: stored elements between rows.  KC: `rows` rows may be read (indexes beyond are clamped: the caller masks what they give),
// and every row holds k up to the last step, zero beyond the true k.  KM: `rows` k may be read (clamped likewise; the OTHER operand is zero
// there), `cols` stored elements per row (a multiple of 8; chunks beyond are clamped, the caller masks what they give).
struct Operand {
  const bf16_t* p;
  int64_t ld;
  int rows;
  int cols;
};

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <int BM_, int BN_, int WM_, int WN_, int PL_, int NST_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, PL = PL_, NST = NST_;
  static constexpr int THREADS = 64 * WM * WN;
  static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;   // 16x16 products of a wave
  static constexpr int KSTEP = PL == 1 ? 64 : 32;
  static constexpr int ROWB = PL == 3 ? 192 : 128;             // bytes of a KC row in a step
  static constexpr int A_BYTES = BM * ROWB, B_BYTES = BN * ROWB, STAGE = A_BYTES + B_BYTES;
  static constexpr int LDS = NST * STAGE;
  static_assert(A_BYTES % (16 * THREADS) == 0 && B_BYTES % (16 * THREADS) == 0, "whole DMA pieces");
  static_assert(LDS <= 163840, "LDS of a CU");
};

// chunk permutation of a KM row: the 16 rows that one transposed read touches ({0..3} + 8 l4) go to different banks
template <int ROW_BYTES>
__device__ __forceinline__ int km_swz(int row) {
  if constexpr (ROW_BYTES % 256 == 0) return (row & 3) | ((row >> 1) & 4);
  else return ((row >> 1) & 1) | ((row >> 2) & 2);
}
template <int PL>
__device__ __forceinline__ int kc_swz(int row) { return PL == 3 ? (row >> 2) & 3 : (row >> 1) & 7; }

// stages one operand's part of a step: R rows (KC) or columns (KM) of the tile
template <class S, int R, int KIND>
struct Stager {
  static constexpr int CH = KIND == KC ? S::ROWB / 16 : R * S::PL / 8;   // 16-B chunks per LDS row
  static constexpr int PIECES = R * S::ROWB / (16 * S::THREADS);
  const char* base;       // uniform
  uint32_t off[PIECES];   // per lane, bytes
  int64_t step;           // bytes per K step
  int64_t ldb;
  int krow0, krows;       // KM: first k row of this lane's pieces is row(j); k rows of the operand

  __device__ __forceinline__ void init(const Operand& o, int r0, int k0) {
    const int tid = threadIdx.x;
    ldb = o.ld * 2;
    if constexpr (KIND == KC) {
      base = reinterpret_cast<const char*>(o.p + (int64_t)r0 * o.ld + (int64_t)k0 * S::PL);
      step = S::ROWB;
      const int last = o.rows - 1 - r0;
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        const int ci = j * S::THREADS + tid, row = ci / CH, c = (ci % CH) ^ kc_swz<S::PL>(row);
        off[j] = (uint32_t)min(row, last) * (uint32_t)ldb + c * 16;
      }
    } else {
      base = reinterpret_cast<const char*>(o.p + (int64_t)k0 * o.ld + (int64_t)r0 * S::PL);
      step = S::KSTEP * ldb;
      krow0 = k0; krows = o.rows;
      const int last = (o.cols - r0 * S::PL) / 8 - 1;
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        const int ci = j * S::THREADS + tid, row = ci / CH, c = (ci % CH) ^ (km_swz<CH * 16>(row) << 1);
        off[j] = (uint32_t)row * (uint32_t)ldb + min(c, last) * 16;
      }
    }
  }
  // the next step, into `dst` (uniform)
  __device__ __forceinline__ void next(char* dst) {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (KIND == KC || krow0 + S::KSTEP <= krows) {
#pragma unroll
      for (int j = 0; j < PIECES; ++j)
        __builtin_amdgcn_global_load_lds((gptr_t)(base + off[j]), (lptr_t)(dst + (j * S::THREADS + wave * 64) * 16), 16, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        const int row = (j * S::THREADS + (int)threadIdx.x) / CH;
        const int over = max(row - (krows - 1 - krow0), 0);   // rows past the last one read the last one
        __builtin_amdgcn_global_load_lds((gptr_t)(base + off[j] - over * ldb), (lptr_t)(dst + (j * S::THREADS + wave * 64) * 16), 16, 0, 0);
      }
    }
    base += step;
    if constexpr (KIND == KM) krow0 += S::KSTEP;
  }
};

// the 16 rows (columns) `g16` of the operand's tile, k slice or plane f
template <class S, int R, int KIND>
__device__ __forceinline__ bf16x8 fragment(const char* img, int g16, int f, int l16, int l4) {
  if constexpr (KIND == KC) {
    const int c = (f * 4 + l4) ^ kc_swz<S::PL>(l16);   // g16 * 16 does not change the permutation
    return *reinterpret_cast<const bf16x8*>(img + (g16 * 16 + l16) * S::ROWB + c * 16);
  } else {
    constexpr int RB = R * S::PL * 2;
    const int blk = S::PL == 1 ? g16 : (g16 >> 1) * (2 * S::PL) + f * 2 + (g16 & 1);
    const int row = (S::PL == 1 ? f * 32 : 0) + 8 * l4 + (l16 >> 2);
    const int at = row * RB + ((blk ^ km_swz<RB>(8 * l4 + (l16 >> 2))) * 32) + (l16 & 3) * 8;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_t)(img + at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_t)(img + at + 4 * RB));
    const s16x8 v = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    return *reinterpret_cast<const bf16x8*>(&v);
  }
}

// acc[mt][nt][q] += C[m = m0 + (wm MT + mt) 16 + l16][n = n0 + (wn NT + nt) 16 + 4 l4 + q], k steps [kt0, kt0 + nk).
// Every thread of the workgroup calls it; smem is free again when it returns.
template <class S, int KA, int KB>
__device__ __forceinline__ void run(const Operand& a, const Operand& b, int m0, int n0, int kt0, int nk, char* smem,
                                    f32x4 (&acc)[S::MT][S::NT]) {
  constexpr int D = S::NST - 1;
  Stager<S, S::BM, KA> sa;
  Stager<S, S::BN, KB> sb;
  constexpr int OPS = Stager<S, S::BM, KA>::PIECES + Stager<S, S::BN, KB>::PIECES;
  static_assert(OPS * (D > 1 ? D - 1 : 0) < 64, "vmcnt range");
  sa.init(a, m0, kt0 * S::KSTEP);
  sb.init(b, n0, kt0 * S::KSTEP);
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
  for (int s = 0; s < D; ++s)
    if (s < nk) { sa.next(smem + s * S::STAGE); sb.next(smem + s * S::STAGE + S::A_BYTES); }
  int slot = 0;
  for (int kt = 0; kt < nk; ++kt) {
    const int ahead = min(D - 1, nk - 1 - kt);   // younger steps in flight
    if (D > 2 && ahead >= 2) wait_vm<(D > 2 ? 2 * OPS : 0)>();
    else if (D > 1 && ahead >= 1) wait_vm<(D > 1 ? OPS : 0)>();
    else wait_vm<0>();
    __builtin_amdgcn_s_barrier();   // step kt is in LDS for everybody; everybody has read step kt - 1
    asm volatile("" ::: "memory");
    if (kt + D < nk) {
      int ps = slot + D;
      if (ps >= S::NST) ps -= S::NST;
      sa.next(smem + ps * S::STAGE);
      sb.next(smem + ps * S::STAGE + S::A_BYTES);
    }
    const char* ia = smem + slot * S::STAGE;
    const char* ib = ia + S::A_BYTES;
    constexpr int NF = S::PL == 1 ? 2 : S::PL;
    if constexpr (S::PL == 1) {
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        bf16x8 fa[S::MT], fb[S::NT];
#pragma unroll
        for (int t = 0; t < S::NT; ++t) fb[t] = fragment<S, S::BN, KB>(ib, wn * S::NT + t, f, l16, l4);
#pragma unroll
        for (int t = 0; t < S::MT; ++t) fa[t] = fragment<S, S::BM, KA>(ia, wm * S::MT + t, f, l16, l4);
#pragma unroll
        for (int x = 0; x < S::MT; ++x)
#pragma unroll
          for (int y = 0; y < S::NT; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[y], fa[x], acc[x][y], 0, 0, 0);
      }
    } else {
      // the planes of one side stay in registers, the other side's pass by in groups of rows
      bf16x8 fb[NF][S::NT];
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int t = 0; t < S::NT; ++t) fb[f][t] = fragment<S, S::BN, KB>(ib, wn * S::NT + t, f, l16, l4);
#pragma unroll
      for (int x = 0; x < S::MT; ++x) {
        bf16x8 fa[NF];
#pragma unroll
        for (int f = 0; f < NF; ++f) fa[f] = fragment<S, S::BM, KA>(ia, wm * S::MT + x, f, l16, l4);
#pragma unroll
        for (int s = NF - 1; s >= 0; --s)   // plane pairs i + j = s, the smallest products first
#pragma unroll
          for (int i = 0; i <= s; ++i)
#pragma unroll
            for (int y = 0; y < S::NT; ++y)
              acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[s - i][y], fa[i], acc[x][y], 0, 0, 0);
      }
    }
    if (++slot == S::NST) slot = 0;
  }
  __syncthreads();
}

template <class S>
__device__ __forceinline__ void clear(f32x4 (&acc)[S::MT][S::NT]) {
#pragma unroll
  for (int x = 0; x < S::MT; ++x)
#pragma unroll
    for (int y = 0; y < S::NT; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// Workgroup -> tile.  Workgroups with equal blockIdx % 8 share an XCD and its L2: each XCD takes one contiguous run of tiles,
// walked in bands of 8 row tiles so that the operand panels in use at a time stay few.
__device__ __forceinline__ void tile_of(int id, int tm, int tn, int& im, int& in) {
  const int total = tm * tn, q = total >> 3, r = total & 7, x = id & 7;
  const int t = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (id >> 3);
  const int band = 8 * tn, first = t / band * 8, in_band = t % band, h = min(8, tm - first);
  im = first + in_band % h;
  in = in_band / h;
}

// x as PL bf16 planes
template <int PL>
__device__ __forceinline__ void split(float x, float (&pl)[PL]) {
#pragma unroll
  for (int p = 0; p < PL; ++p) {
    pl[p] = bf2f(f2bf(x));
    if (p + 1 < PL) x -= pl[p];
  }
  // an infinity minus itself is no rest
  if constexpr (PL > 1) {
    if (__builtin_isinf(pl[0])) {
#pragma unroll
      for (int p = 1; p < PL; ++p) pl[p] = 0.f;
    }
  }
}

// four consecutive elements (e % 4 == 0) of a row, as planes
template <int PL>
__device__ __forceinline__ void store4(bf16_t* row, int64_t e, const float (&v)[4]) {
  float pl[4][PL];
#pragma unroll
  for (int q = 0; q < 4; ++q) split<PL>(v[q], pl[q]);
  bf16_t* at = row + (e >> 5) * (32 * PL) + (e & 31);
#pragma unroll
  for (int p = 0; p < PL; ++p)
    *reinterpret_cast<uint2*>(at + p * 32) = make_uint2(pack_bf16x2(pl[0][p], pl[1][p]), pack_bf16x2(pl[2][p], pl[3][p]));
}
template <int PL>
__device__ __forceinline__ void load4(const bf16_t* row, int64_t e, float (&v)[4]) {
  const bf16_t* at = row + (e >> 5) * (32 * PL) + (e & 31);
#pragma unroll
  for (int q = 0; q < 4; ++q) v[q] = 0.f;
#pragma unroll
  for (int p = PL - 1; p >= 0; --p) {
    const uint2 w = *reinterpret_cast<const uint2*>(at + p * 32);
    v[0] += bf2f(w.x & 0xffff); v[1] += bf2f(w.x >> 16);
    v[2] += bf2f(w.y & 0xffff); v[3] += bf2f(w.y >> 16);
  }
}

}  // namespace tg
