// One output tile of  C[m][n] = sum_k A[m][k] B[n][k]  on the matrix cores, for the training operators (vocab_loss.hip,
// orthogonal.hip).  Only the K loop lives here; the caller's kernel owns the accumulators and its epilogue.
//
// Numbers.  An operand is stored as PL bf16 PLANES whose sum is the value: one plane is a plain bf16 matrix, two planes leave a
// rest of at most 2^-17 |x|, three of 2^-26 |x| (an fp32 value's own half step is 2^-24).  Products of bf16 are exact in fp32.  The plane
// pairs (i, j) with i + j < PL are multiplied -- 1, 3 or 6 MFMAs per product; the pairs left out are below 2^-16 |x y| (two planes)
// and 2^-24 |x y| (three).  The matrix cores run 16 bf16 MFMAs in the time of one fp32 MFMA of the same shape, so six bf16
// products are 2.6 times the rate of native fp32.
//
// Layouts.  The planes of a matrix are interleaved along its contiguous direction in runs of 32: element e, plane p is stored
// at (e / 32) * 32 * PL + p * 32 + e % 32.  One K step then moves the same bytes whatever PL is (64 k of one plane, 32 k of two
// or three), and one plane is the ordinary row-major layout.  An operand is read either way round:
//   KC  rows are m (or n), k contiguous: fragments by ds_read_b128, 8 consecutive k of a row per lane;
//   KM  rows are k, m (or n) contiguous: fragments by ds_read_b64_tr_b16 (the LDS transposes 4 x 16 blocks on the way to the
//       registers), so that no operand needs a transposed copy in memory (two KM operands are slower than one, though: the loss makes
//       a transposed copy of its features where a product would have two).
// LDS images are filled by LDS-DMA, 16 B per lane, lane-linear; bank conflicts are avoided by permuting the 16-B chunks of a
// row on the source address and again on the read.
#pragma once
#include "common.h"
#include <atomic>
#include <type_traits>

namespace tg {

typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4* lds_tr_t;

enum { KC = 0, KM = 1 };

// ld: stored elements between rows.  KC: `rows` rows exist (rows beyond read as zero), and every row holds k up to the last step, zero
// beyond the true k.  KM: `rows` k exist (rows beyond read as zero), `cols` stored elements per row may be read (a multiple of 8; chunks
// beyond are clamped, the caller masks what they give).  A tile's rows, or a step's, span less than 4 GiB.
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

// KG > 1: KG groups of WM x WN waves share the K loop of one tile, each with LDS slots of its own, and add up at the end (in the order of the groups).
// A small tile's step is a chain of latencies -- barrier, LDS, products -- that more waves on the CU hide and more groups shorten.
template <int BM_, int BN_, int WM_, int WN_, int PL_, int NST_, int KG_ = 1>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, PL = PL_, NST = NST_, KG = KG_;
  static constexpr int THREADS = 64 * WM * WN, WG_THREADS = THREADS * KG;   // of a group, of the workgroup
  static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;   // 16x16 products of a wave
  static constexpr int KSTEP = PL == 1 ? 64 : 32;
  static constexpr int ROWB = PL == 3 ? 192 : 128;             // bytes of a KC row in a step
  static constexpr int A_BYTES = BM * ROWB, B_BYTES = BN * ROWB, STAGE = A_BYTES + B_BYTES;
  static constexpr int SLOTS = NST * STAGE, LDS = KG * SLOTS;
  static_assert(A_BYTES % (16 * THREADS) == 0 && B_BYTES % (16 * THREADS) == 0, "whole DMA pieces");
  static_assert(LDS <= 163840, "LDS of a CU");
  static_assert(KG == 1 || BM * BN * 4 <= SLOTS, "the groups' sums pass through the slots");
  // this thread within its group; its wave there; its group (uniform)
  __device__ static __forceinline__ int tid() { return KG == 1 ? (int)threadIdx.x : (int)threadIdx.x % THREADS; }
  __device__ static __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) % (WM * WN); }
  __device__ static __forceinline__ int group() { return KG == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) / (WM * WN); }
  // whether this wave holds the finished 16x16 product (x, y) of its part of the tile; PAIRS: products 2j and 2j + 1 of a row block have one owner
  template <bool PAIRS = false>
  __device__ static __forceinline__ bool owns(int x, int y) { return KG == 1 || (PAIRS ? x * ((NT + 1) / 2) + y / 2 : x * NT + y) % KG == group(); }
};

// chunk permutation of a KM row: the 16 rows that one transposed read touches ({0..3} + 8 l4) go to different banks
template <int ROW_BYTES>
__device__ __forceinline__ int km_swz(int row) {
  if constexpr (ROW_BYTES % 256 == 0) return (row & 3) | ((row >> 1) & 4);
  else return ((row >> 1) & 1) | ((row >> 2) & 2);
}
template <int PL>
__device__ __forceinline__ int kc_swz(int row) { return PL == 3 ? (row >> 2) & 3 : (row >> 1) & 7; }

// stages one operand's part of a step: R rows (KC) or columns (KM) of the tile, by buffer loads to LDS, whose bounds check gives the zeros
// beyond the operand's rows without a branch in the loop
template <class S, int R, int KIND>
struct Stager {
  static constexpr int CH = KIND == KC ? S::ROWB / 16 : R * S::PL / 8;   // 16-B chunks per LDS row
  static constexpr int PIECES = R * S::ROWB / (16 * S::THREADS);
  uint64_t base;          // uniform: the step's first byte
  int64_t left, step;     // bytes of the operand from there on; bytes between steps
  uint32_t off[PIECES];   // per lane, bytes
  int valid;              // steps of this group that exist; further ones read as zero

  __device__ __forceinline__ void init(const Operand& o, int r0, int k0, int steps) {
    const int tid = S::tid();
    valid = steps;
    const int64_t ldb = o.ld * 2;
    if constexpr (KIND == KC) {
      base = (uint64_t)(o.p + (int64_t)r0 * o.ld + (int64_t)k0 * S::PL);
      left = (int64_t)(o.rows - r0) * ldb - (int64_t)k0 * S::PL * 2;
      step = S::ROWB;
    } else {
      base = (uint64_t)(o.p + (int64_t)k0 * o.ld + (int64_t)r0 * S::PL);
      left = (int64_t)(o.rows - k0) * ldb - (int64_t)r0 * S::PL * 2;
      step = S::KSTEP * ldb;
    }
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int ci = j * S::THREADS + tid, row = ci / CH;
      int c;
      if constexpr (KIND == KC) c = (ci % CH) ^ kc_swz<S::PL>(row);
      else c = min((ci % CH) ^ (km_swz<CH * 16>(row) << 1), (o.cols - r0 * S::PL) / 8 - 1);
      off[j] = (uint32_t)row * (uint32_t)ldb + c * 16;
    }
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc() const {
    const uint32_t n = (S::KG > 1 && valid <= 0) || left < 0 ? 0u : left > 0xffffffffll ? 0xffffffffu : (uint32_t)left;
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, n, 0x00027000);
  }
  __device__ __forceinline__ void piece(__amdgpu_buffer_rsrc_t r, int j, char* dst) const {   // dst: uniform
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr_t)(dst + (j * S::THREADS + S::wave() * 64) * 16), 16, off[j], 0, 0, 0);
  }
  __device__ __forceinline__ void advance() { base += step; left -= step; if (S::KG > 1) --valid; }
  __device__ __forceinline__ void next(char* dst) {   // the whole step
    const __amdgpu_buffer_rsrc_t r = rsrc();
#pragma unroll
    for (int j = 0; j < PIECES; ++j) piece(r, j, dst);
    advance();
  }
};

// The compiler drains the DMA queue (vmcnt 0) in front of a transposed LDS read unless the read carries alias information; `restrict` on
// an inlined parameter gives it some.  What orders these reads after the DMA that fills their slot are the loop's own waits and barriers.
__device__ __forceinline__ s16x4 read_tr(lds_tr_t __restrict__ p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p); }

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
    const s16x4 lo = read_tr((lds_tr_t)(img + at));
    const s16x4 hi = read_tr((lds_tr_t)(img + at + 4 * RB));
    const s16x8 v = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    return *reinterpret_cast<const bf16x8*>(&v);
  }
}

// K loop with a ring of NST > 2 slots, for small tiles: NST - 1 steps in flight, one barrier a step.
template <class S, int KA, int KB>
__device__ __forceinline__ void run_ring(Stager<S, S::BM, KA>& sa, Stager<S, S::BN, KB>& sb, int nk, char* smem, f32x4 (&acc)[S::MT][S::NT]) {
  constexpr int D = S::NST - 1, OPS = Stager<S, S::BM, KA>::PIECES + Stager<S, S::BN, KB>::PIECES, NF = S::PL == 1 ? 2 : S::PL;
  static_assert(D >= 2 && OPS * 2 < 64, "vmcnt range");
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = S::wave(), wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
  for (int s = 0; s < D; ++s)
    if (s < nk) { sa.next(smem + s * S::STAGE); sb.next(smem + s * S::STAGE + S::A_BYTES); }
  int slot = 0;
  for (int kt = 0; kt < nk; ++kt) {
    const int ahead = min(D - 1, nk - 1 - kt);   // younger steps in flight
    if (ahead >= 2) wait_vm<2 * OPS>();
    else if (ahead >= 1) wait_vm<OPS>();
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
    bf16x8 fa[NF][S::MT], fb[NF][S::NT];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
#pragma unroll
      for (int t = 0; t < S::NT; ++t) fb[f][t] = fragment<S, S::BN, KB>(ib, wn * S::NT + t, f, l16, l4);
#pragma unroll
      for (int t = 0; t < S::MT; ++t) fa[f][t] = fragment<S, S::BM, KA>(ia, wm * S::MT + t, f, l16, l4);
    }
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j)
        if (S::PL == 1 ? i == j : i + j < S::PL)
#pragma unroll
          for (int x = 0; x < S::MT; ++x)
#pragma unroll
            for (int y = 0; y < S::NT; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j][y], fa[i][x], acc[x][y], 0, 0, 0);
    if (++slot == S::NST) slot = 0;
  }
}

// K loop for large tiles: two slots, and the fragments of the next products read while the present ones multiply.
//
// A step is 2 (one plane), 3 or 6 PHASES; a phase multiplies the fragments it holds, row block by row block, and between the row
// blocks issues the LDS reads of what the next phases need.  The last reads of a slot belong to the last phase but one; then comes the
// step's one barrier (the next step has landed: its DMA went out a whole step earlier; everybody's reads of this slot are done), and
// the last phase issues the DMA of the step after next into the slot, piece by piece between its products: issued in one go the
// pieces stall every wave of the CU at once for about a third of the step.
// Measured on 8192 x 2048 x 8192, one plane, 256 x 256 tiles: 1060 TFLOP/s with DMA, reads and products in turn, 1380 this way
// (KM operands 1130 - 1210); products alone, with nothing to load, 1720, the rate at which the card's power limit holds the clock.
template <class S, int KA, int KB>
__device__ __forceinline__ void run_phased(Stager<S, S::BM, KA>& sa, Stager<S, S::BN, KB>& sb, int nk, char* smem, f32x4 (&acc)[S::MT][S::NT]) {
  constexpr int MT = S::MT, NT = S::NT, NPA = Stager<S, S::BM, KA>::PIECES, NP = NPA + Stager<S, S::BN, KB>::PIECES;
  static_assert(S::NST == 2 && NP < 64, "two slots");
  typedef bf16x8 FA[MT];
  typedef bf16x8 FB[NT];
  const int lane = threadIdx.x & 63, l16 = lane & 15, l4 = lane >> 4;
  const int wave = S::wave(), wm = wave / S::WN, wn = wave % S::WN;
  auto read_a = [&](FA& f, int t, const char* img, int plane) { f[t] = fragment<S, S::BM, KA>(img, wm * MT + t, plane, l16, l4); };
  auto read_b = [&](FB& f, int t, const char* img, int plane) { f[t] = fragment<S, S::BN, KB>(img + S::A_BYTES, wn * NT + t, plane, l16, l4); };
  // products of (a, b), and of what follows: na from plane pa if WA, nb from plane pb if WB, both of image `img`; DMA into `dst`
  auto phase = [&](const FA& a, const FB& b, auto wa, FA& na, int pa, auto wb, FB& nb, int pb, const char* img, auto dma, char* dst) {
    constexpr int RB = decltype(wb)::value ? NT : 0, R = RB + (decltype(wa)::value ? MT : 0);
    __amdgpu_buffer_rsrc_t ra, rb;
    if constexpr (decltype(dma)::value) { ra = sa.rsrc(); rb = sb.rsrc(); }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < MT; ++x) {
      if constexpr (decltype(dma)::value) {
#pragma unroll
        for (int j = x * NP / MT; j < (x + 1) * NP / MT; ++j) {
          if (j < NPA) sa.piece(ra, j, dst);
          else sb.piece(rb, j - NPA, dst + S::A_BYTES);
        }
      }
#pragma unroll
      for (int i = x * R / MT; i < (x + 1) * R / MT; ++i) {
        if (i < RB) read_b(nb, i, img, pb);
        else read_a(na, i - RB, img, pa);
      }
#pragma unroll
      for (int y = 0; y < NT; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[y], a[x], acc[x][y], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (decltype(dma)::value) { sa.advance(); sb.advance(); }
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  auto meet = [&]() {
    wait_vm<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  sa.next(smem); sb.next(smem + S::A_BYTES);
  if (nk > 1) {
    sa.next(smem + S::STAGE); sb.next(smem + S::STAGE + S::A_BYTES);
    wait_vm<NP>();
  } else {
    wait_vm<0>();
  }
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  // The order of a step's products lets the next step start in the same registers as this one.  The reads that a last step makes for the
  // step after it find what lies in the other slot; nothing uses them.
  FA a0, a1;
  FB b0, b1;
  auto first = [&](FB& fb, int pb) {
#pragma unroll
    for (int t = 0; t < NT; ++t) read_b(fb, t, smem, pb);
#pragma unroll
    for (int t = 0; t < MT; ++t) read_a(a0, t, smem, 0);
  };
  auto all = [&](auto step) {
    int kt = 0;
    for (; kt + 2 < nk; ++kt) step(smem + (kt & 1) * S::STAGE, smem + (~kt & 1) * S::STAGE, yes);
    for (; kt < nk; ++kt) step(smem + (kt & 1) * S::STAGE, smem + (~kt & 1) * S::STAGE, no);
  };
  if constexpr (S::PL == 1) {   // "planes" 0 and 1 are the two halves of the 64 k
    first(b0, 0);
    all([&](char* cur, char* nxt, auto dma) {
      phase(a0, b0, yes, a1, 1, yes, b1, 1, cur, no, cur);
      meet();
      phase(a1, b1, yes, a0, 0, yes, b0, 0, nxt, dma, cur);
    });
  } else if constexpr (S::PL == 2) {
    first(b1, 1);
    all([&](char* cur, char* nxt, auto dma) {
      phase(a0, b1, no, a1, 0, yes, b0, 0, cur, no, cur);
      phase(a0, b0, yes, a1, 1, no, b1, 0, cur, no, cur);
      meet();
      phase(a1, b0, yes, a0, 0, yes, b1, 1, nxt, dma, cur);
    });
  } else {
    FA a2;
    FB b2;
    first(b2, 2);
    all([&](char* cur, char* nxt, auto dma) {
      phase(a0, b2, no, a1, 0, yes, b1, 1, cur, no, cur);
      phase(a0, b1, no, a1, 0, yes, b0, 0, cur, no, cur);
      phase(a0, b0, yes, a1, 1, no, b2, 0, cur, no, cur);
      phase(a1, b1, yes, a2, 2, no, b2, 0, cur, no, cur);
      phase(a1, b0, no, a0, 0, no, b2, 0, cur, no, cur);
      meet();
      phase(a2, b0, yes, a0, 0, yes, b2, 2, nxt, dma, cur);
    });
  }
}

template <class S, int KA, int KB>
__device__ __forceinline__ void run_groups(const Operand& a, const Operand& b, int m0, int n0, int kt0, int nk, char* smem, f32x4 (&acc)[S::MT][S::NT]) {
  Stager<S, S::BM, KA> sa;
  Stager<S, S::BN, KB> sb;
  const int each = (nk + S::KG - 1) / S::KG, g = S::group(), own = min(each, nk - g * each);
  sa.init(a, m0, (kt0 + g * each) * S::KSTEP, own);
  sb.init(b, n0, (kt0 + g * each) * S::KSTEP, own);
  char* slots = smem + g * S::SLOTS;
  if constexpr (S::NST == 2) run_phased<S, KA, KB>(sa, sb, each, slots, acc);
  else run_ring<S, KA, KB>(sa, sb, each, slots, acc);
  __syncthreads();
}

// acc[mt][nt][q] += C[m = m0 + (wm MT + mt) 16 + l16][n = n0 + (wn NT + nt) 16 + 4 l4 + q], k steps [kt0, kt0 + nk), nk >= 1; with several
// groups, in the products that the wave owns.  Every thread of the workgroup calls it; smem is free again when it returns.
template <class S, int KA, int KB, bool PAIRS = false>
__device__ __forceinline__ void run(const Operand& a, const Operand& b, int m0, int n0, int kt0, int nk, char* smem, f32x4 (&acc)[S::MT][S::NT]) {
  run_groups<S, KA, KB>(a, b, m0, n0, kt0, nk, smem, acc);
  if constexpr (S::KG > 1) {
    f32x4* mine = reinterpret_cast<f32x4*>(smem + S::group() * S::SLOTS);   // [wave][product][lane]
    const int at = S::wave() * S::MT * S::NT * 64 + (threadIdx.x & 63);
#pragma unroll
    for (int x = 0; x < S::MT; ++x)
#pragma unroll
      for (int y = 0; y < S::NT; ++y) mine[at + (x * S::NT + y) * 64] = acc[x][y];
    __syncthreads();
#pragma unroll
    for (int x = 0; x < S::MT; ++x)
#pragma unroll
      for (int y = 0; y < S::NT; ++y) {
        if (!S::template owns<PAIRS>(x, y)) continue;
        f32x4 v = *reinterpret_cast<const f32x4*>(smem + (at + (x * S::NT + y) * 64) * 16);
#pragma unroll
        for (int k = 1; k < S::KG; ++k) v += *reinterpret_cast<const f32x4*>(smem + k * S::SLOTS + (at + (x * S::NT + y) * 64) * 16);
        acc[x][y] = v;
      }
    __syncthreads();
  }
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

// x as PL bf16 planes; an infinity has no rest (inf - inf) -- unless FINITE, where it becomes NaN
template <int PL, bool FINITE = false>
__device__ __forceinline__ void split(float x, float (&pl)[PL]) {
  pl[0] = bf2f(f2bf(x));
#pragma unroll
  for (int p = 1; p < PL; ++p) {
    x = !FINITE && __builtin_isinf(pl[0]) ? 0.f : x - pl[p - 1];
    pl[p] = bf2f(f2bf(x));
  }
}

// four consecutive elements (e % 4 == 0) of a row, as planes
template <int PL, bool FINITE = false>
__device__ __forceinline__ void store4(bf16_t* row, int64_t e, const float (&v)[4]) {
  float pl[4][PL];
#pragma unroll
  for (int q = 0; q < 4; ++q) split<PL, FINITE>(v[q], pl[q]);
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

// Eight consecutive elements of a row as one 16-B store per plane: the products y and y + 1 of a row block hold, per lane, four elements of each
// (v0, v1); neighbouring rows of lanes swap so that a lane has eight of one.  e: the first element of product y in the row (a
// multiple of 16); a row's two products (32 elements) then go out as 64 contiguous bytes per plane instead of four pieces of 8 bytes twice.
// Every lane of the wave calls it; `live` lanes' rows are written.
template <int PL, bool FINITE = false>
__device__ __forceinline__ void store_pair(bf16_t* row, int64_t e, const float (&v0)[4], const float (&v1)[4], int l4, bool live) {
  float p0[4][PL], p1[4][PL];
#pragma unroll
  for (int q = 0; q < 4; ++q) { split<PL, FINITE>(v0[q], p0[q]); split<PL, FINITE>(v1[q], p1[q]); }
  const int64_t at = e + (l4 & 1) * 16 + (l4 >> 1) * 8;
  bf16_t* dst = row + (at >> 5) * (32 * PL) + (at & 31);
#pragma unroll
  for (int p = 0; p < PL; ++p) {
    const auto a = __builtin_amdgcn_permlane16_swap(pack_bf16x2(p0[0][p], p0[1][p]), pack_bf16x2(p1[0][p], p1[1][p]), false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(pack_bf16x2(p0[2][p], p0[3][p]), pack_bf16x2(p1[2][p], p1[3][p]), false, false);
    if (live) *reinterpret_cast<uint4*>(dst + p * 32) = make_uint4(a[0], b[0], a[1], b[1]);
  }
}

// A kernel may take more LDS than the default: asked for once per kernel, again if that failed.  Threads that come at the same time each ask, for the
// same value.
template <typename K>
int allow_lds(K kernel, int bytes, std::atomic<bool>& done) {
  if (done.load(std::memory_order_acquire)) return SGPO_OK;
  SGPO_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.store(true, std::memory_order_release);
  return SGPO_OK;
}
#define ALLOW(kernel, bytes)                                           \
  do {                                                                 \
    static std::atomic<bool> done_{false};                             \
    if (const int rc_ = tg::allow_lds(kernel, bytes, done_)) return rc_; \
  } while (0)

}  // namespace tg
