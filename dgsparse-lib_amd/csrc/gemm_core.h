// gemm_core.h -- tiled matrix product on the matrix cores of gfx950, the core of the gated feed-forward block and the 8-bit product.
//
//   C[m, n] = sum over k of A(m, k) B(n, k)
//
// An operand lies in memory either K-inner (row m holds its K values side by side) or K-outer (row k holds the M values side by side, as
// in the gradients); neither is ever transposed in memory.  A workgroup of WM x WN waves makes a BM x BN tile of C, 128 bytes of K a step:
//   * global -> LDS by the buffer unit (16 bytes a lane, no registers in between), two LDS buffers, the next step's loads in flight while
//     this step's matrix instructions run.  Rows and K values behind the matrix read as zeros (their lanes ask for an offset behind the
//     descriptor's range).
//   * LDS -> registers: 16 bytes a lane = 16 rows x 64 bytes of K ("slice") for one 16 x 16 x (64 bytes) matrix step.  K-inner tiles are
//     read with ds_read_b128, K-outer tiles with the transposing ds_read_b64_tr_b16.
//   * The 16-byte pieces of an LDS row are permuted (XOR with some bits of the row), so that the rows that are read together lie in
//     different banks; the loads fetch the pieces in that order, the LDS side of a load being a straight line by construction.
//   * The operands enter the matrix instruction as (B, A): a lane then holds four neighbouring n of one row m, which leave in one store.
// 32-bit operands take another way to LDS (Gemm3 below): through registers, where each value becomes three of 16 bits.
// Sums are held in 32 bits throughout; K is walked in order, so a result depends on the tile shape and the number of splits alone, and
// these on the sizes alone.
#pragma once
#include <type_traits>

#include "dense_common.h"

namespace dgs {

struct fp8 { uint8_t v; };  // e4m3 (the OCP form: bias 7, no infinities)

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kStepBytes = 128;        // of K, a step
constexpr uint32_t kNowhere = 0x80000000u;  // an offset behind every descriptor's range: reads as zero (and so does anything up to 2^31 behind it)
constexpr int kRange = 0x7ffffff0;     // the descriptors' range: offsets within a tile stay below it (checked by the dispatch)

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) char lds_char;

// 16 bytes of K for each of 16 rows (per lane: one row, 16 bytes): one step of the matrix cores over 64 bytes of K
union Slice {
  dgs_u4 u;
  bf16x8 b;
  f16x8 h;
  float f[4];
  s16x4 s[2];
};
// acc[i][j] += a[i] b[j] over the slice.  32 bits: lane group g holds k = 4 g .. 4 g + 3, and the q-th of four instructions takes the q-th
// of them; the four go round all sums, so that none waits for the one before.
template <typename T, int FM, int FN>
__device__ __forceinline__ void multiply(const Slice (&a)[FM], const Slice (&b)[FN], f32x4 (&acc)[FM][FN]) {
#pragma unroll
  for (int q = 0; q < (sizeof(T) == 4 ? 4 : 1); q++)
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) {
        if constexpr (sizeof(T) == 4)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[j].f[q], a[i].f[q], acc[i][j], 0, 0, 0);
        else if constexpr (std::is_same<T, f16>::value)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[j].h, a[i].h, acc[i][j], 0, 0, 0);
        else
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j].b, a[i].b, acc[i][j], 0, 0, 0);
      }
}

// ---- one operand's tile in LDS: R rows (of M or N) x 128 bytes of K, R * 128 bytes -------------------------------------------------
template <typename T, int R, bool KO>
struct Tile {
  static_assert(sizeof(T) == 2 || (sizeof(T) == 1 && !KO), "32-bit operands: Planes");
  static constexpr int kBytes = R * kStepBytes;
  static constexpr int kK = kStepBytes / (int)sizeof(T);       // K values a step
  static constexpr int kCpr = KO ? R * (int)sizeof(T) / 16 : 8;  // 16-byte pieces of an LDS row (K-outer: a row is one k)

  // which piece of the row the LDS place `slot` holds (and the other way round): rows that are read together go to different banks
  static __device__ __forceinline__ int mix(int row, int slot) {
    if constexpr (!KO) return slot ^ ((row >> 1) & 7);
    else return slot ^ (2 * (((row & 3) + ((row >> 1) & 4)) & (kCpr / 2 - 1)));  // (4 rows and every second 8 rows are read together)
  }
  // A thread loads pieces id, id + THREADS, ... (of R * 8, in LDS order): kRowsPerLoad rows apart, at the same place of the row where the
  // permutation does not change over that distance (kSame).
  // offset(): of piece `id` from the tile's corner; K-outer: kNowhere where the piece lies behind the row's `left` bytes (rows behind the
  // matrix are behind the descriptor's range for either kind).  k: its first K value in the step (K-inner).
  static __device__ __forceinline__ uint32_t offset(int id, int64_t ld, int64_t left, int &k) {
    const int row = id / kCpr, piece = mix(row, id % kCpr);
    k = piece * (16 / (int)sizeof(T));
    return !KO || piece * 16 < left ? (uint32_t)(row * (int)ld + piece * 16) : kNowhere;
  }
  template <int THREADS>
  static constexpr bool same() {
    return THREADS / kCpr % 16 == 0;
  }
  // the slice of rows [16 i, 16 i + 16), 64 bytes kk of K
  static __device__ __forceinline__ void read(const char *lds, int row0, int kk, int lane, Slice &s) {
    if constexpr (!KO) {
      const int row = row0 + (lane & 15), slot = mix(row, (lane >> 4) + 4 * kk);
      s.u = *reinterpret_cast<const dgs_u4 *>(lds + row * kStepBytes + slot * 16);
    } else {
      // each 16 lanes read 4 k x 16 m (8 bytes a lane) and get them transposed: a lane has the 4 k of its m
      const int i = lane & 15;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int k = 32 * kk + 8 * (lane >> 4) + 4 * h + (i >> 2);
        const int byte = row0 * 2 + (i & 3) * 8;
        const char *p = lds + k * (kCpr * 16) + mix(k, byte / 16) * 16 + byte % 16;
        s.s[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds_char *)p);
      }
    }
  }
};

// What a launch multiplies.  Leading dimensions in bytes.  `pair`: how the second pointers are used:
//   kOne     C[0] = A[0] B[0]
//   kDual    the tile's columns come in halves from B[0] and B[1] (BN / 2 columns each): C0 = A[0] B[0], C1 = A[0] B[1]
//   kSum     C[0] = A[0] B[0] + A[1] B[1]   (one walk over K after the other)
//   kTwo     C[0] = A[0] B[0], C[1] = A[1] B[0]  (workgroups for one, then for the other)
enum Pair { kOne, kDual, kSum, kTwo };
struct GemmArgs {
  const char *A[2], *B[2];
  int64_t lda, ldb;
  int64_t M, N, K;  // N: of one matrix (kDual: columns of C0)
  int tiles_m, tiles_n, splits;
};

// Which tile a workgroup makes.  Workgroups go round the 8 XCDs, each with an L2 of its own: XCD x takes the x-th eighth of the tiles, in
// panels of kPanel tile rows, so that the tiles that run together on an XCD share their rows of A and columns of B there.
constexpr int kXcds = 8, kPanel = 8;
struct Where { int m, n, z; };
__device__ __forceinline__ Where where_of(int tiles_m, int tiles_n) {
  const int total = tiles_m * tiles_n;
  int b = (int)blockIdx.x;
  const int each = total / kXcds, rest = total % kXcds, x = b % kXcds;
  b = b / kXcds + x * each + (x < rest ? x : rest);
  const int panel = b / (kPanel * tiles_n), in = b % (kPanel * tiles_n);
  const int rows = tiles_m - panel * kPanel < kPanel ? tiles_m - panel * kPanel : kPanel;
  return {panel * kPanel + in % rows, in / rows, (int)blockIdx.y};
}

// bytes from a tile's corner to the matrix's last row's end, as a descriptor's range
__device__ __forceinline__ int tile_range(int64_t rows, int64_t ld) {
  const int64_t b = rows * ld;
  return b < kRange ? (int)b : kRange;
}
// The workgroup's waves meet: this wave's LDS accesses are done, loads to registers may be on their way.
__device__ __forceinline__ void lds_meet() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// How a workgroup's waves share a tile
template <int BM, int BN, int WM, int WN, int PAIR>
struct Shares {
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static constexpr int kCols = PAIR == kDual ? BN / 2 : BN;  // columns of C that a tile covers
  // column of the tile's B rows where the wave's j-th 16 columns begin, and the column of C
  static __device__ __forceinline__ int b_row(int wn, int j) {
    if constexpr (PAIR == kDual) return (j < FN / 2 ? 0 : BN / 2) + wn * (BN / 2 / WN) + 16 * (j % (FN / 2));
    return wn * (BN / WN) + 16 * j;
  }
  static __device__ __forceinline__ int c_col(int wn, int j) {
    if constexpr (PAIR == kDual) return wn * (BN / 2 / WN) + 16 * (j % (FN / 2));
    return wn * (BN / WN) + 16 * j;
  }
};

// The tile's sums: acc[i][j] = 16 x 16 at rows 16 i, columns col_of(j) of the wave's part; lane l register r holds m = l % 16, n = 4 (l / 16) + r.
// (The 8-bit product keeps its own walk over K, with a scale behind each 128 bytes: fp8_kernel.)
template <typename T, int BM, int BN, int WM, int WN, bool A_KO, bool B_KO, int PAIR>
struct Gemm : Shares<BM, BN, WM, WN, PAIR> {
  using S = Shares<BM, BN, WM, WN, PAIR>;
  using S::FM, S::FN, S::b_row, S::kThreads, S::kWaves;
  using TA = Tile<T, BM, A_KO>;
  using TB = Tile<T, BN, B_KO>;
  static constexpr int QA = BM * 8 / kThreads, QB = BN * 8 / kThreads;  // 16-byte loads of a thread a step
  static_assert(QA * kThreads == BM * 8 && QB * kThreads == BN * 8, "whole loads");
  static_assert(PAIR != kDual || (!B_KO && QB % 2 == 0), "halves of the loads");

  // One thread's share of a step's loads: the offset of the first, and of the others where they do not follow from it by the rows' distance.
  static constexpr bool kSameA = TA::template same<kThreads>(), kSameB = TB::template same<kThreads>();
  static constexpr int PB = PAIR == kDual ? QB / 2 : QB;  // loads of one B (kDual: both alike)
  struct Load {
    uint32_t a[kSameA ? 1 : QA], b[kSameB ? 1 : PB];
    int ka, kb;
    int da, db;  // kSame: bytes from one load's row to the next one's (the same in every lane)
  };
  static __device__ __forceinline__ void plan(Load &l, const GemmArgs &g, int m0, int n0) {
    const int64_t left_a = ((g.M - m0) * (int64_t)sizeof(T) + 15) / 16 * 16, left_b = ((g.N - n0) * (int64_t)sizeof(T) + 15) / 16 * 16;
    int k;
#pragma unroll
    for (int q = 0; q < (kSameA ? 1 : QA); q++) {
      l.a[q] = TA::offset(q * kThreads + (int)threadIdx.x, g.lda, left_a, k);
      if (q == 0) l.ka = k;
    }
#pragma unroll
    for (int q = 0; q < (kSameB ? 1 : PB); q++) {
      l.b[q] = TB::offset(q * kThreads + (int)threadIdx.x, g.ldb, left_b, k);
      if (q == 0) l.kb = k;
    }
    l.da = kThreads / TA::kCpr * (int)g.lda;
    l.db = kThreads / TB::kCpr * (int)g.ldb;
  }
  // The loads of step s (of `steps` a walk over K; kSum: 2 * steps in all) into one LDS buffer
  static __device__ __forceinline__ void load(const Load &l, const GemmArgs &g, int m0, int n0, int s, int steps, int z, char *la, char *lb) {
    const int seg = PAIR == kSum ? (s >= steps ? 1 : 0) : 0;
    const int st = s - seg * steps;
    const int64_t k0 = (int64_t)st * TA::kK, kleft = g.K - k0;
    const int left = (int)(kleft < TA::kK ? kleft : TA::kK);  // K values of this step
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    {
      const char *p = g.A[PAIR == kTwo ? z : seg] + (A_KO ? k0 * g.lda + m0 * (int64_t)sizeof(T) : m0 * g.lda + k0 * (int64_t)sizeof(T));
      const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), 0, tile_range(A_KO ? kleft : g.M - m0, g.lda), 0x00027000);
      const bool on = A_KO || l.ka < left;
#pragma unroll
      for (int q = 0; q < QA; q++) {
        const uint32_t o = kSameA ? l.a[0] + (uint32_t)(q * l.da) : l.a[kSameA ? 0 : q];
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)(lds_char *)(la + (q * kWaves + wave) * 1024), 16, on ? (int)o : (int)kNowhere, 0, 0, 0);
      }
    }
#pragma unroll
    for (int half = 0; half < (PAIR == kDual ? 2 : 1); half++) {
      const char *p = g.B[PAIR == kDual ? half : seg] + (B_KO ? k0 * g.ldb + n0 * (int64_t)sizeof(T) : n0 * g.ldb + k0 * (int64_t)sizeof(T));
      const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), 0, tile_range(B_KO ? kleft : g.N - n0, g.ldb), 0x00027000);
      const bool on = B_KO || l.kb < left;
#pragma unroll
      for (int q = 0; q < PB; q++) {
        const uint32_t o = kSameB ? l.b[0] + (uint32_t)(q * l.db) : l.b[kSameB ? 0 : q];
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)(lds_char *)(lb + ((half * PB + q) * kWaves + wave) * 1024), 16, on ? (int)o : (int)kNowhere, 0, 0, 0);
      }
    }
  }
  static __device__ __forceinline__ void compute(const char *la, const char *lb, int wm, int wn, int lane, f32x4 (&acc)[FM][FN]) {
#pragma unroll
    for (int kk = 0; kk < 2; kk++) {
      __builtin_amdgcn_sched_barrier(0);  // (one half's operands in registers at a time)
      Slice a[FM], b[FN];
#pragma unroll
      for (int j = 0; j < FN; j++) TB::read(lb, b_row(wn, j), kk, lane, b[j]);
#pragma unroll
      for (int i = 0; i < FM; i++) TA::read(la, wm * (BM / WM) + 16 * i, kk, lane, a[i]);
      multiply<T>(a, b, acc);
    }
  }
};

// This wave's loads have landed in LDS and its LDS reads are done; then the workgroup's.  (Said outright: a barrier alone need not wait for
// loads that go to LDS.)
__device__ __forceinline__ void loads_done() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// The main loop, 16-bit types: steps [s0, s1) into acc.  The four LDS buffers are separate arrays, so that the compiler sees that
// a step's reads and the next step's loads do not meet and does not wait for the loads in between.
#define DGS_GEMM_LDS(G)                                              \
  __shared__ __align__(16) char ldsA0[G::TA::kBytes], ldsB0[G::TB::kBytes]; \
  __shared__ __align__(16) char ldsA1[G::TA::kBytes], ldsB1[G::TB::kBytes];

template <typename G>
__device__ __forceinline__ void gemm_loop(const GemmArgs &g, int m0, int n0, int s0, int s1, int steps, int z, char *ldsA0, char *ldsB0,
                                          char *ldsA1, char *ldsB1, int wm, int wn, int lane, f32x4 (&acc)[G::FM][G::FN]) {
#pragma unroll
  for (int i = 0; i < G::FM; i++)
#pragma unroll
    for (int j = 0; j < G::FN; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (s0 >= s1) return;
  typename G::Load l;
  G::plan(l, g, m0, n0);
  G::load(l, g, m0, n0, s0, steps, z, ldsA0, ldsB0);
  loads_done();
  int s = s0;
  for (; s + 1 < s1; s += 2) {  // (no way out in the middle: the sums would be moved between registers there)
    G::load(l, g, m0, n0, s + 1, steps, z, ldsA1, ldsB1);
    G::compute(ldsA0, ldsB0, wm, wn, lane, acc);
    loads_done();
    if (s + 2 < s1) G::load(l, g, m0, n0, s + 2, steps, z, ldsA0, ldsB0);
    G::compute(ldsA1, ldsB1, wm, wn, lane, acc);
    loads_done();
  }
  if (s < s1) G::compute(ldsA0, ldsB0, wm, wn, lane, acc);
}

// ---- 32-bit operands ----------------------------------------------------------------------------------------------------------
// A 32-bit value as three of 16 bits (bf16: 8 bits of mantissa each, the range of 32 bits): x = hi + mid + lo but for 2^-27 x, each rounded to
// nearest from what is left.  A product of two such values is six products of their parts, the ones below 2^-26 of it left out: as close
// as a product rounded to 32 bits, on matrix instructions that take the six (96 cycles for 16 x 16 x 32) in less than half the time of the
// 32-bit ones (256).  The parts' products are exact, their sums held in 32 bits.  What differs: an infinity becomes a NaN (inf - inf).
//
// What is left of a value is one instruction, the dot product of its pair's parts with (-1, 0) or (0, -1) added to it: exact, like the
// subtraction it stands for, without the part widened to 32 bits first (7 instructions a pair for the three parts, not 11).  The constants
// are kept in registers: as inline constants these instructions take them for both halves.  The pair's other value enters such a product as 0
// times it, which an infinity or a NaN makes a NaN: right where the two lie in one row (K-inner: the row has the value either way), wrong where
// they lie in two (K-outer, ALONE: dW's row of a good gradient beside a bad one).  There each value is widened and subtracted by itself.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
struct Minus {  // (-1, 0) and (0, -1) in bf16
  uint32_t lo = 0x0000bf80u, hi = 0xbf800000u;
  __device__ __forceinline__ Minus() { asm volatile("" : "+s"(lo), "+s"(hi)); }
};
template <bool ALONE>
__device__ __forceinline__ void split3(f32x2 r, const Minus &minus, uint32_t (&part)[3]) {
#pragma unroll
  for (int q = 0; q < 3; q++) {
    const bf16x2 h = __builtin_convertvector(r, bf16x2);
    part[q] = __builtin_bit_cast(uint32_t, h);
    if (q < 2 && ALONE) {
      r[0] -= (float)h[0];
      r[1] -= (float)h[1];
    } else if (q < 2) {
      r[0] = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, minus.lo), r[0], false);
      r[1] = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, minus.hi), r[1], false);
    }
  }
}

// One operand's step of 32 K values in LDS: three planes of R rows x 64 bytes (K-inner) or 32 rows x 2 R bytes (K-outer).
template <int R, bool KO>
struct Planes {
  static constexpr int kPlane = R * 64, kBytes = 3 * kPlane;
  static constexpr int kPieces = KO ? R / 4 : 8;  // 16-byte pieces (4 values) of a row in memory
  using Outer = Tile<bf16, R, true>;
  static __device__ __forceinline__ uint32_t offset(int id, int64_t ld, int64_t left, int &k) {
    const int row = id / kPieces, piece = id % kPieces;
    k = KO ? 0 : 4 * piece;
    return !KO || piece * 16 < left ? (uint32_t)(row * (int)ld + piece * 16) : kNowhere;
  }
  static __device__ __forceinline__ int mix(int row, int slot) {
    if constexpr (KO) return Outer::mix(row, slot);
    else return slot ^ (-(row >> 2) & 3);  // (the 16 lanes that read together take rows 0-3, 12-15 of one piece and 4-7, 8-11 of the next)
  }
  // piece `id` of the step (4 neighbouring values), split, into the planes
  static __device__ __forceinline__ void write(char *lds, int id, const f32x4 &x, const Minus &minus) {
    const int row = id / kPieces, piece = id % kPieces;
    uint32_t p[2][3];
#pragma unroll
    for (int h = 0; h < 2; h++) split3<KO>(f32x2{x[2 * h], x[2 * h + 1]}, minus, p[h]);
    char *at = lds + row * (KO ? 2 * R : 64) + mix(row, piece / 2) * 16 + piece % 2 * 8;
#pragma unroll
    for (int q = 0; q < 3; q++) *reinterpret_cast<dgs_u2 *>(at + q * kPlane) = dgs_u2{p[0][q], p[1][q]};
  }
  // The 16 rows at row0, a multiple of 16: lane group g has K values 8 g .. 8 g + 7.  `Place`: where the lane reads of a plane at row 0; row0 is added
  // (K-outer: a bit of the place within the LDS row, which the permutation leaves as it is, or turns: an exclusive or).
  struct Place { uint32_t at[KO ? 2 : 1]; };
  static __device__ __forceinline__ Place place(int lane) {
    Place p;
    if constexpr (!KO) {
      p.at[0] = (lane & 15) * 64 + mix(lane & 15, lane >> 4) * 16;
    } else {
      const int i = lane & 15;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int k = 8 * (lane >> 4) + 4 * h + (i >> 2);
        p.at[h] = k * 2 * R + mix(k, (i & 3) / 2) * 16 + (i & 1) * 8;
      }
    }
    return p;
  }
  static __device__ __forceinline__ void read(const char *plane, const Place &p, int row0, Slice &s) {
    if constexpr (!KO) {
      s.u = *reinterpret_cast<const dgs_u4 *>(plane + p.at[0] + row0 * 64);
    } else {
#pragma unroll
      for (int h = 0; h < 2; h++)
        s.s[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds_char *)(plane + (p.at[h] ^ (row0 * 2))));
    }
  }
};

template <int BM, int BN, int WM, int WN, bool A_KO, bool B_KO, int PAIR>
struct Gemm3 : Shares<BM, BN, WM, WN, PAIR> {
  using S = Shares<BM, BN, WM, WN, PAIR>;
  using S::FM, S::FN, S::b_row, S::kThreads;
  static constexpr int kK = 32;
  using PA = Planes<BM, A_KO>;
  using PB = Planes<BN, B_KO>;
  static constexpr int QA = BM * 8 / kThreads, QB = BN * 8 / kThreads, PBQ = PAIR == kDual ? QB / 2 : QB;  // (as in Gemm)
  static_assert(kThreads % PA::kPieces == 0 && kThreads % PB::kPieces == 0, "a thread's pieces lie below each other");
  struct Raw { f32x4 a[QA], b[QB]; };
  struct Load { uint32_t a, b; int ka, kb; };
  static __device__ __forceinline__ void load(const Load &l, const GemmArgs &g, int m0, int n0, int s, int steps, int z, Raw &raw) {
    const int seg = PAIR == kSum ? (s >= steps ? 1 : 0) : 0;
    const int64_t k0 = (int64_t)(s - seg * steps) * kK, kleft = g.K - k0;
    const int left = (int)(kleft < kK ? kleft : kK);
    {
      const char *p = g.A[PAIR == kTwo ? z : seg] + (A_KO ? k0 * g.lda + m0 * (int64_t)4 : m0 * g.lda + k0 * (int64_t)4);
      const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), 0, tile_range(A_KO ? kleft : g.M - m0, g.lda), 0x00027000);
      const bool on = A_KO || l.ka < left;
#pragma unroll
      for (int q = 0; q < QA; q++)
        raw.a[q] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, on ? (int)(l.a + (uint32_t)(q * (kThreads / PA::kPieces) * (int)g.lda)) : (int)kNowhere, 0, 0));
    }
#pragma unroll
    for (int half = 0; half < (PAIR == kDual ? 2 : 1); half++) {
      const char *p = g.B[PAIR == kDual ? half : seg] + (B_KO ? k0 * g.ldb + n0 * (int64_t)4 : n0 * g.ldb + k0 * (int64_t)4);
      const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), 0, tile_range(B_KO ? kleft : g.N - n0, g.ldb), 0x00027000);
      const bool on = B_KO || l.kb < left;
#pragma unroll
      for (int q = 0; q < PBQ; q++)
        raw.b[half * PBQ + q] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, on ? (int)(l.b + (uint32_t)(q * (kThreads / PB::kPieces) * (int)g.ldb)) : (int)kNowhere, 0, 0));
    }
  }
  // Steps [s0, s1) into acc.  The next step's operands are on their way to registers while this one's, split, are multiplied out of LDS: each
  // value is split once for the workgroup, not by each of the two waves that read it (169343 x 128 x 512, forward and backward: 1316 -> 1182 us),
  // and one buffer of 48 KB leaves room for three workgroups on a CU, which fill each other's waits at the two barriers of a step.
  static __device__ __forceinline__ void run(const GemmArgs &g, int m0, int n0, int s0, int s1, int steps, int z, char *lds, int wm, int wn, int lane, f32x4 (&acc)[FM][FN]) {
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (s0 >= s1) return;
    const Minus minus;
    const typename PA::Place placeA = PA::place(lane);
    const typename PB::Place placeB = PB::place(lane);
    const int t = (int)threadIdx.x;
    Load l;
    l.a = PA::offset(t, g.lda, ((g.M - m0) * 4 + 15) / 16 * 16, l.ka);
    l.b = PB::offset(t, g.ldb, ((g.N - n0) * 4 + 15) / 16 * 16, l.kb);
    Raw raw;
    load(l, g, m0, n0, s0, steps, z, raw);
    char *la = lds, *lb = lds + PA::kBytes;
    for (int s = s0; s < s1; s++) {
      lds_meet();  // (the step before has been read)
#pragma unroll
      for (int q = 0; q < QA; q++) PA::write(la, q * kThreads + t, raw.a[q], minus);
#pragma unroll
      for (int q = 0; q < QB; q++) PB::write(lb, q * kThreads + t, raw.b[q], minus);
      load(l, g, m0, n0, s + 1 < s1 ? s + 1 : s, steps, z, raw);  // (the last step's again, unused: a branch round the loads is slower, 1205 us for 1185)
      lds_meet();
      Slice b[FN][3];
#pragma unroll
      for (int j = 0; j < FN; j++)
#pragma unroll
        for (int q = 0; q < 3; q++) PB::read(lb + q * PB::kPlane, placeB, b_row(wn, j), b[j][q]);
#pragma unroll
      for (int i = 0; i < FM; i++) {
        Slice a[3];
#pragma unroll
        for (int q = 0; q < 3; q++) PA::read(la + q * PA::kPlane, placeA, wm * (BM / WM) + 16 * i, a[q]);
        constexpr int pa[6] = {0, 2, 1, 0, 1, 0}, pb[6] = {2, 0, 1, 1, 0, 0};  // the small ones first
#pragma unroll
        for (int q = 0; q < 6; q++)
#pragma unroll
          for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j][pb[q]].b, a[pa[q]].b, acc[i][j], 0, 0, 0);
      }
    }
  }
};

// ---- few rows of A: the rows of B on their way to a wave's matrix instructions ---------------------------------------------------------
// A wave loads 16 rows x 128 bytes in two loads of 8 whole lines: neighbouring lanes take neighbouring 16 bytes (16 rows x 64 bytes a load, as the
// instruction wants them, reads 45 MB at 4.6 TB/s, these at 5.7), and turns them by way of 2 KB of LDS of its own into the two slices.
// Only this wave touches them, and a wave's LDS accesses are made in their order: no barrier, only the compiler is held.
struct Lines {
  dgs_u4 u[2];
};
__device__ __forceinline__ void turn(char *lds, int lane, const Lines &x, Slice (&s)[2]) {
  using L = Tile<bf16, 16, false>;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int row = 8 * h + (lane >> 3);
    *reinterpret_cast<dgs_u4 *>(lds + row * kStepBytes + L::mix(row, lane & 7) * 16) = x.u[h];
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int kk = 0; kk < 2; kk++) L::read(lds, 0, kk, lane, s[kk]);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// four neighbouring columns of a row; `vec`: the row's stride and base allow one store
template <typename T>
__device__ __forceinline__ void store4(T *p, const f32x4 &v, int64_t left, bool vec) {
  if (vec && left >= 4) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4 *>(p) = v;
    } else {
      union { dgs_u2 u; T t[4]; } x;
#pragma unroll
      for (int k = 0; k < 4; k++) x.t[k] = from_f32<T>(v[k]);
      *reinterpret_cast<dgs_u2 *>(p) = x.u;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (k < left) p[k] = from_f32<T>(v[k]);
  }
}
template <typename T>
__device__ __forceinline__ f32x4 load4(const T *p, int64_t left, bool vec) {
  f32x4 v;
  if (vec && left >= 4) {
    if constexpr (sizeof(T) == 4) {
      v = *reinterpret_cast<const f32x4 *>(p);
    } else {
      union { dgs_u2 u; T t[4]; } x;
      x.u = *reinterpret_cast<const dgs_u2 *>(p);
#pragma unroll
      for (int k = 0; k < 4; k++) v[k] = to_f32(x.t[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = k < left ? to_f32(p[k]) : 0.0f;
  }
  return v;
}

// Rows of another stride than the 16-byte loads take: copied once, padded with zeros to a multiple of 16 bytes.
template <typename T>
__global__ __launch_bounds__(kBlock) void pad_rows_kernel(int64_t rows, int64_t cols, const T *__restrict__ src, int64_t ld, int64_t ldo, T *__restrict__ dst) {
  const int64_t t = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  const int64_t per = ldo * (int64_t)sizeof(T) / 16, row = t / per, c = t % per * (16 / (int64_t)sizeof(T));
  if (row >= rows) return;
  union { dgs_u4 u; T t[16 / sizeof(T)]; } x;
  x.u = dgs_u4{0u, 0u, 0u, 0u};
#pragma unroll
  for (int k = 0; k < 16 / (int)sizeof(T); k++)
    if (c + k < cols) x.t[k] = src[row * ld + c + k];
  *reinterpret_cast<dgs_u4 *>(dst + row * ldo + c) = x.u;
}
template <typename T>
static int pad_rows(int64_t rows, int64_t cols, const void *src, int64_t ld, int64_t ldo, void *dst, hipStream_t st) {
  const int64_t n = rows * (ldo * (int64_t)sizeof(T) / 16), blocks = (n + kBlock - 1) / kBlock;
  if (!grid_ok(blocks)) return DGS_ERANGE;
  hipLaunchKernelGGL((pad_rows_kernel<T>), dim3((unsigned)blocks), dim3(kBlock), 0, st, rows, cols, (const T *)src, ld, ldo, (T *)dst);
  return check_launch();
}
inline bool rows16(const void *p, int64_t cols, int64_t ld, size_t size) {
  return aligned_to(p, 16) && (cols * (int64_t)size) % 16 == 0 && (ld * (int64_t)size) % 16 == 0;
}

// C[e] = the splits' sums in their order
template <typename T>
__global__ __launch_bounds__(kBlock) void join_splits_kernel(int64_t count, int splits, const float *__restrict__ partial, T *__restrict__ c0, T *__restrict__ c1, int64_t each) {
  const int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (e >= count) return;
  float s = 0.0f;
#pragma unroll 4
  for (int z = 0; z < splits; z++) s += partial[z * count + e];
  if (e < each) c0[e] = from_f32<T>(s); else c1[e - each] = from_f32<T>(s);
}

// ---- which tile, how many splits ------------------------------------------------------------------------------------------
// kBig: 256 x 256, 8 waves, a workgroup a CU; kMid: 128 x 128, 4 waves, 2 a CU; kSmall: 64 x 64, 4 waves.  A larger tile reads less from L2
// and LDS for a product, but there have to be enough of them, and they must not lie half beside the matrix: the largest whose tiles (times
// splits of K, where the caller can split) fill three quarters of the CUs and cover at most a quarter more than the next smaller ones.
enum Shape { kBig, kMid, kSmall };
struct TilePlan { Shape shape; int tiles_m, tiles_n, splits; };
static TilePlan tile_plan(int64_t M, int64_t N, int64_t steps, int mats, bool dual, bool big, bool split) {
  TilePlan p = {kSmall, 0, 0, 1};
  const int sizes[] = {256, 128, 64};
  const int64_t cus = cu_count(), want = cus * 3 / 4;
  for (int s = big ? kBig : kMid; s <= kSmall; s++) {
    const int64_t tm = (M + sizes[s] - 1) / sizes[s], cols = dual ? sizes[s] / 2 : sizes[s], tn = (N + cols - 1) / cols, tiles = tm * tn * mats;
    if (s < kSmall) {
      const int64_t half = sizes[s] / 2, least = ((M + half - 1) / half) * ((N + cols / 2 - 1) / (cols / 2));  // in quarters of this tile
      if (4 * tm * tn > least + least / 4) continue;
    }
    p.shape = (Shape)s;
    p.tiles_m = (int)tm;
    p.tiles_n = (int)tn;
    p.splits = 1;
    if (tiles >= want) break;
    if (split) {
      const int64_t fill = (2 * cus + tiles - 1) / tiles, most = steps / (s == kSmall ? 4 : 16);
      p.splits = (int)(fill < most ? fill : most < 1 ? 1 : most);
      if (tiles * p.splits >= want) break;
    }
  }
  return p;
}

}  // namespace dgs
