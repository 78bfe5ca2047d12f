// spmm_impl.h -- CSR SpMM (sum / max / min / mean + arg ids) for gfx950.
//
// Replaces csrspmm_seqreduce_rowbalance_kernel (reference include/cuda/spmm_cuda.cuh:10-55), which maps ONE
// THREAD to one (row, feature), re-reads col/val through L1 once per feature and walks every row - however
// long - sequentially in one thread.  Power-law graphs (a few rows with 10^4..10^5 nnz) stall that schedule,
// and short rows pay three dependent memory latencies (rowptr -> col -> B) per handful of nnz.
//
// Schedule used here (all wave64, plan-free: the only state is a caller-provided scratch workspace):
//
//   feature mapping   a row of the output is owned by a GROUP of G lanes, each lane holding V=4 consecutive
//                     features: one B row = G coalesced dwordx4 loads (N=64: 16 lanes x 16 B = one 256-B row,
//                     so a single wave-level load instruction gathers 4 different B rows = 1 KiB).
//
//   K0 spmm_classify  one pass over rowptr: every LONG row (len > T1) is cut into units of <= CH nnz, appended
//                     to a unit table in the workspace (block-level scan + ONE atomicAdd per block).
//
//   K1 spmm_fused     one launch, two kinds of blocks:
//        unit blocks  persistent, stride over the unit table, one wave per unit: 64 (col,val) pairs at a time
//                     through LDS, the NG=64/G groups take interleaved nnz (G lanes still read one coalesced B
//                     row), up to 8 gathers in flight per lane, partials combined across groups by a fixed
//                     xor-butterfly (ds_bpermute/DPP).  Single-unit rows write C directly, multi-unit rows write
//                     a partial row (slot = unit id) to the workspace.
//        row blocks   one wave per 64 consecutive rows.  rowptr comes in with one coalesced load, the (col,val)
//                     pairs of runs of SHORT rows (len <= T1) are staged into a per-wave LDS tile with coalesced
//                     non-temporal loads, the run's nnz stream is cut into NG nnz-balanced row-aligned pieces
//                     and each group streams its piece through a rolling window of independent B-row gathers,
//                     storing a row of C whenever it meets a row-end flag.  Per-feature accumulation order is
//                     CSR order => bit-identical to algorithm 0 (fmaf chain for sum/mean, single-rounded
//                     products + first-wins ties for max/min).
//
//   K2 spmm_combine   folds the partial rows of every multi-unit row in unit order (fixed tree).
//
//   Determinism: atomics only allocate table slots; every value is produced by a fixed reduction tree, so
//   results are run-to-run identical.  max/min carry (value, column id, position) so that the first occurrence
//   in CSR order wins ties under any split => values and E bit-exact vs algorithm 0 for every row length.
//   sum/mean: sequential (bit-exact) for rows <= T1, fixed-tree (<= 1e-5 rel) above.
//
//   Measured on MI355X (profiles/): the fused kernel is bound by the L2-miss path (~6.5 TB/s of 128-B fabric
//   reads at a ~30% L2 hit rate on the 1M x 1M power-law graph); see DESIGN.md for the ladder that led here.
//
//   spmm_small: inputs up to 2^18 nnz / 2^16 rows take ONE launch (row blocks only, long rows reduced in place).
//
//   spmm_panel (spmm_panel.h): dense graphs whose dense operand overflows the L2s take a column-panel sweep with the
//   accumulators resident in LDS instead of K1's row blocks (panel_plan() below decides; rows longer than 4096 nnz
//   still go through K0 -> unit blocks -> K2).  MIN over NaN products is order-dependent: the split paths detect it
//   and redo the affected elements sequentially (seq_redo).
#pragma once
#include <stdlib.h>

#include <atomic>

#include "dgs_common.h"
#include "spmm_panel.h"

namespace dgs {


// ---------------------------------------------------------------------------------------------------------
// tuning constants
#ifndef DGS_XCD_REMAP
#define DGS_XCD_REMAP 1
#endif
#ifndef DGS_T1
#define DGS_T1 64
#endif
#ifndef DGS_T2
#define DGS_T2 DGS_T1
#endif
#ifndef DGS_CAP
#define DGS_CAP 512
#endif
constexpr int kT1 = DGS_T1;   // rows up to this many nnz are streamed sequentially by one group (row blocks)
constexpr int kT2 = DGS_T2;   // rows in (T1, T2] would be reduced in place by the wave that owns their row block; the
                              // measured optimum is T2 == T1 (every row > T1 becomes units: better balance), so that
                              // in-place path is live only in spmm_small, where it handles ALL long rows
#ifndef DGS_TRACE
#define DGS_TRACE 0
#endif
#if DGS_TRACE
__device__ unsigned long long *g_dgs_trace = nullptr;  // [wave][8] timestamps (experiment: per-wave timeline)
#define DGS_TS(k) do { if (g_dgs_trace && lane == 0 && blockIdx.y == 0) g_dgs_trace[(size_t)trace_id * 8 + (k)] = wall_clock64(); } while (0)
#else
#define DGS_TS(k) do { } while (0)
#endif
constexpr int kCap = DGS_CAP; // (col,val) pairs per wave LDS tile of the row blocks (4 KiB per wave, 16 KiB per block)
constexpr int kRowsPerWave = 64;
#ifndef DGS_KU1
#define DGS_KU1 6
#endif
constexpr int kU1 = DGS_KU1;   // rolling window of B-row gathers per lane in the row stream
#ifndef DGS_KU
#define DGS_KU 8
#endif
constexpr int kU = DGS_KU;     // gathers in flight per lane in the wave-cooperative unit loop

struct SpmmWs {       // workspace header (zeroed every call)
  int n_units;        // K0 -> fused/K2: number of unit descriptors
  int n_pslots;       // partial-row slots handed out (multi-unit rows only)
  int arrivals;       // spmm_panel: panel steps finished, summed over workgroups (soft barrier)
  int n_long;         // K0 -> K2: number of multi-unit rows (entries of the long-row table)
  int hub[8];         // strict schedule: units per length class of the hub rows (spmm_strict.h)
};

// Unit tables, as the kernels see them.  Two producers: spmm_classify (plan-free call: tables in the workspace, rebuilt
// every call) and the cached plan (spmm_plan.hip: tables built once per matrix, units of hub rows cut at column-slice
// boundaries and sorted by (slice, first column), one slice per XCD).
//   unit     {row, first nnz, nnz in the unit, partial-row slot | -1 when the unit is the whole row}
//   longrow  {row, first partial slot, units in the row, -}           (multi-unit rows only: what spmm_combine folds)
struct UnitTab {
  const int *n_units;
  const int *n_long;
  const int *xcd_start;  // [9] first unit of each XCD's share, or nullptr = equal eighths of the table
  const int4 *units;
  const int4 *longrows;
  const int *xcd_end = nullptr;  // [8] where each XCD's walk stops (a plan's hub-row units are skipped when the hub blocks
                                 // chain those rows), or nullptr = the next share's start
  // In-kernel fold (round 5): long-row index of every partial slot + one arrival counter per long row (zero at launch).  The
  // unit wave that brings a row's count to its number of units folds the row on the spot - no combine launch.  nullptr = the
  // partial rows wait for spmm_combine.
  const int *slot_long = nullptr;
  int *arrive = nullptr;
  unsigned part_bytes = 0;  // bytes of the partial-row region (what the fold's buffer descriptors cover; < 2^31, fold_fits)
  int pstride = 0;          // FOLD twin: floats between two partial rows (fold_stride: whole 128-byte lines); else the rows are N apart
};

struct WsLayout {
  size_t off_units, off_long, off_part, off_parte, off_slot, off_arrive, total;
  int64_t max_units, max_pslots, max_long;
  int ch;
};

// Unit length CH: 256 nnz by default, grown for huge inputs so that the partial-row scratch stays bounded.
static inline int unit_len(int64_t nnz) {
  int ch = 256;
  while ((nnz / ch) > 65536 && ch < (1 << 20)) ch <<= 1;
  return ch;
}

// Row stride of the partial rows when they are folded INSIDE the fused launch: whole 128-byte lines per slot, on a 128-byte aligned
// base, so that no two partial rows ever share a cache line.  The hand-over is write-through sc1 stores -> drain -> counter -> sc1
// loads (MI355X guide, R1 form); what that form does not spell out is what an sc1 load returns for a line its own XCD still holds
// from an EARLIER read - which is exactly what slots narrower than a line would make it do (the folder of row A reads the line that
// also holds the first slot of row B, and folds B later).  With one slot per line(s) every line of a row is read by its folder for
// the first time in the launch, after every writer has drained: the question never arises.  Costs address space only (N = 16: 64 ->
// 128 bytes per slot; the bytes written and read are the same).  The combine launch (fold off) keeps the dense layout.
#ifndef DGS_FOLD_DENSE
#define DGS_FOLD_DENSE 0  // 1 (tests/emu/mutation_check_mem.py only): the twin keeps the combine launch's dense layout - slots narrower than a line share lines
#endif
static inline int64_t fold_stride(int64_t N) { return DGS_FOLD_DENSE ? N : (N + 31) / 32 * 32; }
template <typename T>
static inline T *align128(T *p) { return reinterpret_cast<T *>((reinterpret_cast<uintptr_t>(p) + 127) & ~uintptr_t(127)); }
// feature tiles a launch over N floats can have (16-byte lanes: 256- or, narrowed, 64-float tiles; scalar lanes: 64-float tiles)
static inline int64_t max_tiles(int64_t N) { return (N + 63) / 64 + 1; }
static inline WsLayout ws_layout(int reduce_op, int64_t N, int64_t nnz) {
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  WsLayout L;
  L.ch = unit_len(nnz);
  // sum over long rows of ceil(len/ch) <= nnz/ch + #long rows; the strict schedule (spmm_strict.h) keeps its hub-row units
  // in per-class regions behind nnz/kT1 + 2 front entries: another 2 * nnz/64 + 128 at most (class c holds <= slices * nnz /
  // (threshold << c) entries, slices / threshold <= 1/64)
  L.max_units = 3 * (nnz / kT2) + nnz / L.ch + 160;
  L.max_pslots = 2 * (nnz / L.ch) + 2;               // same sum over rows longer than ch only (they need partials)
  L.max_long = nnz / L.ch + 2;                       // rows longer than ch
  L.off_units = up(sizeof(SpmmWs));
  L.off_long = L.off_units + up((size_t)L.max_units * sizeof(int4));
  L.off_part = L.off_long + up((size_t)L.max_long * sizeof(int4));
  const size_t prow = up((size_t)L.max_pslots * fold_stride(N) * sizeof(float) + 128);  // one partial row per unit of a multi-unit row (fold_stride + alignment slack: either layout fits)
  L.off_parte = L.off_part + prow;
  const bool arg = (reduce_op == DGS_MAX || reduce_op == DGS_MIN);
  L.off_slot = L.off_parte + (arg ? prow : 0);                         // long-row index of every partial slot
  L.off_arrive = L.off_slot + up((size_t)L.max_pslots * sizeof(int));  // arrival counter of every long row
  L.total = L.off_arrive + up((size_t)L.max_long * max_tiles(N) * sizeof(int)) + 256;  // (one counter per row and feature tile)
  return L;
}

// With a cached plan the workspace only holds the partial rows of the multi-unit rows.
// (+ the arrival counters of the in-kernel fold, one int per long row; the slot -> long-row map is part of the plan)
static inline WsLayout ws_layout_plan(int reduce_op, int64_t N, int64_t pslots, int64_t n_long) {
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  WsLayout L{};
  L.max_pslots = pslots;
  L.max_long = n_long;
  L.off_part = 0;
  const size_t prow = up((size_t)(pslots > 0 ? pslots : 1) * fold_stride(N) * sizeof(float) + 128);
  L.off_parte = prow;
  const bool arg = (reduce_op == DGS_MAX || reduce_op == DGS_MIN);
  L.off_arrive = prow + (arg ? prow : 0);
  L.total = L.off_arrive + up((size_t)(n_long > 0 ? n_long : 1) * max_tiles(N) * sizeof(int)) + 256;
  return L;
}
// plan buffer: [256-byte header][column grid: 129 ints][units: max_units int4][long rows: max_long int4]; the capacities
// (and so the offsets) are a pure function of nnz, the actual counts live in the header
constexpr int kPlanCh = 256;          // unit length of the plan's unit table (large inputs)
constexpr int kPlanChMin = 64;        // ... and the shortest one it uses (small inputs)
constexpr int kPlanSliceMin = 128;    // smallest row length that may be cut on the column grid
constexpr int kPlanUnitMin = 16;      // smallest nnz-per-cell target of a cut row
constexpr int kPlanCells = 128;       // finest column grid: 8 slices (one per XCD) x 16 cells
constexpr int kHubChain = 16384;    // default hub threshold of the sum / mean launches (DGS_HUB_CHAIN; 0 = no hub chains)
constexpr int kHubChainMin = 1024;  // smallest threshold accepted (bounds the hub tables: nnz / 1024 rows)
struct PlanLayout {
  int64_t max_units, max_long, max_hub, max_srows;
  size_t off_bounds, off_units, off_long, off_hub, off_slot, off_strict, total;
};
// The strict-order schedule over a plan (round 5): every row longer than T1 as {row, first nnz, nnz, -}, sorted LONGEST FIRST,
// behind a 32-byte header with the sizes of its three length classes - what spmm_classify_strict builds per call otherwise.
struct StrictPlanHdr {
  int n_hub, n_mid, n_whole;  // rows > kStrictHub (one dense table, chained by hub workgroups), > kStrictMid (4 feature slices), the rest
  int pad[5];
};
static inline size_t plan_off_strict(size_t off_slot, int64_t n_pslots) { return off_slot + (((size_t)n_pslots * sizeof(int) + 255) & ~size_t(255)); }
// where the slot -> long-row map sits: behind the hub table (build-time layout: capacities; compact plan: counts)
static inline size_t plan_off_slot(size_t off_hub, int64_t n_hub) { return off_hub + (((size_t)n_hub * sizeof(int4) + 255) & ~size_t(255)); }
static inline PlanLayout plan_layout(int64_t nnz) {
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  PlanLayout L;
  // a cut row of L nnz has at most max(8, L / kPlanUnitMin) cells, each with one ragged unit, plus L / ch full ones
  L.max_units = nnz / kT1 + 8 * (nnz / kPlanSliceMin) + nnz / kPlanUnitMin + nnz / kPlanChMin + 16;
  L.max_long = nnz / kPlanSliceMin + nnz / kPlanChMin + 2;
  L.off_bounds = 256;
  L.off_units = 256 + 768;  // (kPlanCells + 1) ints
  L.max_hub = nnz / kHubChainMin + 16;
  L.off_long = L.off_units + up((size_t)L.max_units * sizeof(int4));
  L.off_hub = L.off_long + up((size_t)L.max_long * sizeof(int4));
  // hub region: max_hub entries {row, first nnz, nnz, -}  (a compact plan: n_hub entries); then one int per partial slot: the
  // index of the slot's row in the long-row table (what the in-kernel fold needs to find the row's arrival counter)
  L.off_slot = plan_off_slot(L.off_hub, L.max_hub);
  L.max_srows = nnz / kT1 + 2;  // rows longer than T1
  L.off_strict = plan_off_strict(L.off_slot, L.max_units);
  L.total = L.off_strict + up(sizeof(StrictPlanHdr) + (size_t)L.max_srows * sizeof(int4)) + 256;
  return L;
}

// ---------------------------------------------------------------------------------------------------------
// cross-group combine helpers (all 64 lanes active)
template <int OP>
__device__ __forceinline__ bool arg_better(float mine, int mypos, float other, int opos) {
  // "other" replaces "mine" iff it wins under first-occurrence-wins semantics of algorithm 0
  if constexpr (OP == DGS_MAX) return (mine < other) || (mine == other && opos < mypos);
  return (mine > other) || (mine == other && opos < mypos);
}

// ei/ep: arg column id and the position of its FIRST strict improvement.  el: position of the LAST time the value
// was (re)assigned - needed only for MIN, whose macro `(acc < t) ? acc : t` takes the LATER operand on a tie, so that
// among equal minima (+0.0 / -0.0 are the only equal floats with different bits) the value of the last one survives
// while E still names the first one.  MAX keeps the earlier operand on a tie, so value and E travel together.
template <int G, int V, int OP>
__device__ __forceinline__ void cross_group_reduce(float (&acc)[V], int (&ei)[V], int (&ep)[V], int (&el)[V]) {
  constexpr bool ARG = (OP == DGS_MAX || OP == DGS_MIN);
#pragma unroll
  for (int m = G; m < 64; m <<= 1) {
#pragma unroll
    for (int v = 0; v < V; v++) {
      const float o = __shfl_xor(acc[v], m, 64);
      if constexpr (ARG) {
        const int oi = __shfl_xor(ei[v], m, 64);
        const int op = __shfl_xor(ep[v], m, 64);
        if constexpr (OP == DGS_MIN) {
          const int ol = __shfl_xor(el[v], m, 64);
          if (acc[v] > o) {
            acc[v] = o;
            ei[v] = oi;
            ep[v] = op;
            el[v] = ol;
          } else if (acc[v] == o) {
            if (op < ep[v]) {
              ei[v] = oi;
              ep[v] = op;
            }
            if (ol > el[v]) {
              acc[v] = o;
              el[v] = ol;
            }
          }
        } else {
          if (arg_better<OP>(acc[v], ep[v], o, op)) {
            acc[v] = o;
            ei[v] = oi;
            ep[v] = op;
          }
        }
      } else {
        acc[v] += o;  // IEEE addition is commutative: both partners compute the same sum => fixed tree
      }
    }
  }
}

// position-tracking reduction step for the split path (pos = CSR position, or unit index in K3)
template <int OP>
__device__ __forceinline__ void reduce_step_pos(float &res, int &eidx, int &epos, int &elast, float w, float x, int c,
                                                int pos) {
  if constexpr (OP == DGS_MAX) {
    const float t = w * x;
    if (res < t) {
      eidx = c;
      epos = pos;
    }
    res = (res < t) ? t : res;
  } else if constexpr (OP == DGS_MIN) {
    const float t = w * x;
    if (res > t) {
      eidx = c;
      epos = pos;
    }
    if (!(res < t)) elast = pos;  // the macro assigns t here (also on ties)
    res = (res < t) ? res : t;
  } else {
    res = __builtin_fmaf(w, x, res);
  }
}

// MIN with NaN products is ORDER-DEPENDENT: `(acc < t) ? acc : t` turns acc into NaN at a NaN product and lets the
// NEXT product replace it unconditionally, so no split of the row can be recombined.  The split paths therefore only
// DETECT the case -- nf[v] = fma(t, 0, nf[v]) goes NaN as soon as one product was NaN (or inf: a false alarm that
// merely takes the slow path) -- and the affected (row, feature) elements are redone as one sequential chain.
constexpr int kNanMark = -2;  // partial-row arg id of an element that met a NaN product (never leaves the workspace)

template <int G, int V>
__device__ __forceinline__ unsigned nan_flags(const float (&nf)[V]) {
  unsigned m = 0;
#pragma unroll
  for (int v = 0; v < V; v++) m |= (nf[v] != nf[v]) ? (1u << v) : 0u;
#pragma unroll
  for (int d = G; d < 64; d <<= 1) m |= (unsigned)__shfl_xor((int)m, d, 64);
  return m;
}

// Virtual columns (accumulating MIN, "around" form - AccArg below, dgsparse.dist): the column ids [lo, lo + n) of the
// matrix do not name rows of the dense operand B but rows of C, the output the launch commits into - the pair (C, E)[row]
// already holds rides through row `row`'s chain as ONE entry (column lo + row, weight 1), at the place its columns have in
// the row; ids >= lo + n are the rows of B shifted by n.  n == 0: plain columns.
struct VirtCols {
  const float *C = nullptr;
  int lo = INT_MAX, n = 0;
};
template <bool VIRT>
__device__ __forceinline__ const float *dense_row(const float *B, const int c, const int N, const VirtCols &vc) {
  if constexpr (!VIRT) {
    return B + (int64_t)c * N;
  } else {
    const bool virt = (unsigned)(c - vc.lo) < (unsigned)vc.n;  // (c < lo wraps to a huge unsigned)
    const float *base = virt ? vc.C : B;
    const int r = virt ? c - vc.lo : (c >= vc.lo ? c - vc.n : c);
    return base + (int64_t)r * N;
  }
}

// Sequential algorithm-0 chain of row [rs,re) for the elements of this lane selected by `mask` (MIN fix-up, rare).
template <int V, int OP, bool VIRT = false>
__device__ __forceinline__ void seq_redo(unsigned mask, int rs, int re, int N, int f0, const int *__restrict__ col,
                                         const float *__restrict__ val, const float *__restrict__ B, float (&acc)[V],
                                         int (&ei)[V], const VirtCols vc = VirtCols{}) {
#pragma unroll
  for (int v = 0; v < V; v++)
    if (mask >> v & 1) {
      acc[v] = reduce_init<OP>();
      ei[v] = -1;
    }
  for (int p = rs; p < re; p++) {
    const int c = col[p];
    const float w = val ? val[p] : 1.0f;
    float x[V];
    load_vec<V>(dense_row<VIRT>(B, c, N, vc) + f0, x);
#pragma unroll
    for (int v = 0; v < V; v++)
      if (mask >> v & 1) reduce_step<OP>(acc[v], ei[v], w, x[v], c);
  }
}

// ---------------------------------------------------------------------------------------------------------
// Hub rows are taken longest first (a 50 k-nnz row is the critical path of the whole call): class c holds the rows with
// kStrictHub << c < nnz <= kStrictHub << (c + 1) (the last class: everything longer), each class has its own region of the
// unit table behind the front entries, sized for the worst case, and the unit waves walk class 5, 4, ... 0, then the front.
constexpr int kHubClasses = 6;
struct HubTab {
  int base[kHubClasses];  // first table entry of each class region (one entry {row, first nnz, nnz, -} per hub row)
  int mid_top;            // strict schedule: the 4-slice units grow down from here (whole-tile units grow up from entry 0)
};
// Regions behind `first` entries; class c holds at most nnz / (thub << c) rows.
static inline HubTab hub_tab(int64_t nnz, int thub, int64_t first) {
  HubTab t;
  int64_t o = first;
  t.mid_top = (int)o;
  for (int c = 0; c < kHubClasses; c++) {
    t.base[c] = (int)o;
    o += nnz / ((int64_t)thub << c) + 16;
  }
  return t;
}
static inline int64_t hub_tab_entries(int64_t nnz, int thub) {  // sum of the class regions: <= 2 nnz / thub + 96
  int64_t o = 0;
  for (int c = 0; c < kHubClasses; c++) o += nnz / ((int64_t)thub << c) + 16;
  return o;
}
__host__ __device__ __forceinline__ int hub_class(int len, int thub) {
  int c = 0;
  while (c < kHubClasses - 1 && len > (thub << (c + 1))) c++;
  return c;
}
// What the hub blocks of a launch walk: per-class row counts (device: the classify pass or the plan wrote them) + the table.
struct HubArg {
  const int *cnt;     // [ncls] rows per class
  const int4 *rows;   // table the class regions of `ht` index
  HubTab ht;
  int ncls;           // kHubClasses (tables of a classify pass), 1 (a plan's table: dense, sorted longest first), 0 = none
};

// ---------------------------------------------------------------------------------------------------------
// K0: scan rowptr once and cut every long row (len > tlong) into units of <= ch nnz; multi-unit rows also get an entry
// of the long-row table (what spmm_combine folds).  Each thread looks at kK0Rows rows, a block-level exclusive scan
// turns the per-thread counts into offsets, and ONE 64-bit atomicAdd per block reserves the block's range of the unit
// table and of the partial slots (same-address atomics cost ~12 ns each when they serialise at L2; per-row atomics
// made this kernel 44 us, per-block ones ~5); blocks that own multi-unit rows add one more for the long-row table.
// Only the position of a row's entries in the tables depends on the atomics, never a value.
constexpr int kK0Rows = 16;
// Rows longer than thub (INT_MAX = none) are not cut at all: they go to the hub table (one entry per row in the region of its
// length class, HubTab) and are chained whole by the hub blocks of the fused launch (spmm_hub_body).
static __global__ __launch_bounds__(kBlock) void spmm_classify(int M, int ch, int tlong, int thub, const HubTab ht,
                                                               const int *__restrict__ rowptr,
                                                               SpmmWs *__restrict__ hdr, int4 *__restrict__ units,
                                                               int4 *__restrict__ longrows, int *__restrict__ slot_long,
                                                               int *__restrict__ arrive, int ntiles) {
  __shared__ int s_wsum[kBlock / kWave], s_psum[kBlock / kWave], s_lsum[kBlock / kWave];
  __shared__ int s_base, s_pbase, s_lbase;
  // block b owns the CONTIGUOUS rows [b*4096, (b+1)*4096): its units form one run of the table that covers
  // neighbouring rows, which is what lets the unit path give each XCD rows that share columns (see spmm_units_body)
  const int nthreads = kBlock;
  const int tid = blockIdx.x * kBlock * kK0Rows + threadIdx.x;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int mine = 0, pmine = 0, lmine = 0;  // units of this thread's rows; units that need a partial slot; multi-unit rows
  unsigned hugemask = 0, hubmask = 0;
#pragma unroll
  for (int i = 0; i < kK0Rows; i++) {
    const int r = i * nthreads + tid;
    if (r < M) {
      const int len = rowptr[r + 1] - rowptr[r];
      if (len > thub) {
        hubmask |= 1u << i;
      } else if (len > tlong) {
        const int nch = (len + ch - 1) / ch;
        mine += nch;
        if (nch > 1) {
          pmine += nch;
          lmine++;
        }
        hugemask |= 1u << i;
      }
    }
  }
  int incl = mine, pincl = pmine, lincl = lmine;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int t = __shfl_up(incl, d, kWave);
    const int tp = __shfl_up(pincl, d, kWave);
    const int tl = __shfl_up(lincl, d, kWave);
    if (lane >= d) {
      incl += t;
      pincl += tp;
      lincl += tl;
    }
  }
  if (lane == kWave - 1) {
    s_wsum[wave] = incl;
    s_psum[wave] = pincl;
    s_lsum[wave] = lincl;
  }
  __syncthreads();
  int woff = 0, total = 0, pwoff = 0, ptotal = 0, lwoff = 0, ltotal = 0;
#pragma unroll
  for (int w = 0; w < kBlock / kWave; w++) {
    if (w < wave) {
      woff += s_wsum[w];
      pwoff += s_psum[w];
      lwoff += s_lsum[w];
    }
    total += s_wsum[w];
    ptotal += s_psum[w];
    ltotal += s_lsum[w];
  }
  if (threadIdx.x == 0) {
    // both counters with ONE 64-bit atomic (n_units low word, n_pslots high word; the header is 16-byte aligned):
    // same-address atomics from all blocks serialise at L2, so one is half the queue of two
    unsigned long long old = 0;
    if (total)
      old = atomicAdd(reinterpret_cast<unsigned long long *>(&hdr->n_units),
                      (unsigned long long)(unsigned)total | ((unsigned long long)(unsigned)ptotal << 32));
    s_base = (int)(unsigned)(old & 0xffffffffull);
    s_pbase = (int)(unsigned)(old >> 32);
    s_lbase = ltotal ? atomicAdd(&hdr->n_long, ltotal) : 0;
  }
  __syncthreads();
  while (hubmask) {  // rare (hundreds in a million rows): one atomicAdd per row on the counter of its length class
    const int i = __ffs((int)hubmask) - 1;
    hubmask &= hubmask - 1;
    const int r = i * nthreads + tid;
    const int rs = rowptr[r], len = rowptr[r + 1] - rs;
    const int c = hub_class(len, thub);
    units[ht.base[c] + atomicAdd(&hdr->hub[c], 1)] = make_int4(r, rs, len, 0);
  }
  if (!mine) return;
  int off = s_base + woff + incl - mine;
  int poff = s_pbase + pwoff + pincl - pmine;
  int loff = s_lbase + lwoff + lincl - lmine;
  while (hugemask) {
    const int i = __ffs((int)hugemask) - 1;
    hugemask &= hugemask - 1;
    const int r = i * nthreads + tid;
    const int rs = rowptr[r], re = rowptr[r + 1];
    const int nch = (re - rs + ch - 1) / ch;
    for (int k = 0; k < nch; k++) {
      const int p0 = rs + k * ch;
      units[off + k] = make_int4(r, p0, min(ch, re - p0), nch > 1 ? poff + k : -1);
      if (nch > 1 && slot_long) slot_long[poff + k] = loff;  // in-kernel fold: which long row a partial slot belongs to
    }
    off += nch;
    if (nch > 1) {
      if (arrive)  // ... and the row's arrival counters, one per feature tile (the workspace's contents are undefined on entry)
        for (int t = 0; t < ntiles; t++) arrive[(int64_t)loff * ntiles + t] = 0;
      longrows[loff++] = make_int4(r, poff, nch, 0);
      poff += nch;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// Wave-cooperative reduction of the nnz range [p0,p1) of one row: 64 (col,val) pairs at a time through the
// wave's LDS tile, the NG groups take interleaved nnz (each B row is still one coalesced G-lane read), up to kU
// gathers in flight per lane.  Leaves per-group partials in acc/ei/ep (combine with cross_group_reduce).
template <int G, int V, int OP, bool HAS_VAL, bool VIRT = false>
__device__ __forceinline__ void coop_accumulate(int p0, int p1, int lane, int g, int f0, bool fl, int N,
                                                const int *__restrict__ col, const float *__restrict__ val,
                                                const float *__restrict__ B, const int *__restrict__ Em, int orow,
                                                int2 *tile, float (&acc)[V], int (&ei)[V], int (&ep)[V],
                                                int (&el)[V], float (&nf)[V], const VirtCols vc = VirtCols{}) {
  constexpr int NG = kWave / G;
  for (int t0 = p0; t0 < p1; t0 += kWave) {
    const int cnt = min(kWave, p1 - t0);
    __builtin_amdgcn_wave_barrier();
    if (lane < cnt) {
      const int c = ld_stream(col + t0 + lane);
      const float w = HAS_VAL ? ld_stream(val + t0 + lane) : 1.0f;
      tile[lane] = make_int2(c, __float_as_int(w));
    }
    __builtin_amdgcn_wave_barrier();
    for (int j = g; j < cnt; j += NG * kU) {
      int c[kU];
      float w[kU];
      float x[kU][V];
      int m[kU][V];
      // tile reads and gathers are issued unconditionally, the entry index clamped into the tile: as conditional blocks each
      // ds_read got an lgkmcnt(0) of its own (8 serial LDS latencies per batch; ISA read, late round 3).  A clamped entry is
      // the batch's last valid one, so the extra gather is a repeat of an address already in flight.
      const int fo = fl ? f0 : 0;
#pragma unroll
      for (int q = 0; q < kU; q++) {
        const int2 cv = tile[min(j + q * NG, cnt - 1)];
        c[q] = cv.x;
        w[q] = __int_as_float(cv.y);
      }
#pragma unroll
      for (int q = 0; q < kU; q++) {
        load_vec_gather<V>(dense_row<VIRT>(B, c[q], N, vc) + fo, x[q]);
        if constexpr (OP == kOpMaskSum) load_vec<V>(Em + (int64_t)c[q] * N + fo, m[q]);
      }
#pragma unroll
      for (int q = 0; q < kU; q++)
        if (j + q * NG < cnt && fl) {
#pragma unroll
          for (int v = 0; v < V; v++) {
            if constexpr (OP == kOpMaskSum) {
              if (m[q][v] == orow) acc[v] = __builtin_fmaf(w[q], x[q][v], acc[v]);
            } else {
              reduce_step_pos<OP>(acc[v], ei[v], ep[v], el[v], w[q], x[q][v], c[q], t0 + j + q * NG);
              if constexpr (OP == DGS_MIN) nf[v] = __builtin_fmaf(w[q] * x[q][v], 0.0f, nf[v]);
            }
          }
        }
    }
  }
}

}  // namespace dgs
#include "spmm_strict.h"
namespace dgs {

// ---------------------------------------------------------------------------------------------------------
// K1: short rows.  Per wave: 64 consecutive rows; runs of short rows are staged into LDS as (col | row-end flag,
// val) pairs; the run's nnz stream is cut into NG nnz-balanced, row-aligned pieces, one per group; each group
// streams its piece U nnz at a time (U independent B-row gathers in flight, no per-row wait) and stores a row
// of C whenever it meets a row-end flag.  Per-feature accumulation order = CSR order (bit-exact vs algorithm 0).
// Also builds the unit table for long rows.
struct RowsLds {
  int2 tile[kBlock / kWave][kCap];
  int4 rows[kBlock / kWave][kRowsPerWave + 1];  // {start, end, next non-empty short row, -}
};

// Accumulating variants (ACC): the row result is merged into what C (and E) already hold instead of overwriting it.
//   sum  C[orow] += result
//   max  (C, E)[orow] = the better of the old pair and (result, arg + col_off), first occurrence winning ties.  The two
//        pairs come from two column subsets of the same matrix rows (dgsparse.dist: columns this rank owns / halo
//        columns), whose ids live in one extended space [0, nl) = local, [nl, ...) = halo slots in global order; h_lo
//        halo slots belong to lower ranks, i.e. come BEFORE the local columns in a row.  key() restores that order, so
//        for rows with sorted columns "smaller key" = "earlier in CSR order" and MAX's rule (the earlier operand keeps
//        value and arg on a tie) is reproduced exactly.
//   min  MIN keeps the LATER operand's value bits on a tie while E names the FIRST minimum, so a pair can be appended to
//        what precedes it in the row or the other way round, but two pairs of interleaved column sets cannot be merged.
//        The caller therefore says where this product's columns lie: h_lo != 0 = they all PRECEDE the columns (C, E)
//        already cover, h_lo == 0 = they all FOLLOW them (dgsparse.dist: the lower-rank halo entries, then the higher-rank
//        ones, in two launches), and the commit is algorithm 0's own step applied to the two pairs in that order.  An
//        output row the earlier products had no entry for holds the empty-row (0, -1); a non-empty MIN result with arg -1
//        can only be the identity, so (arg < 0 and value != identity) marks it and the new pair simply replaces it.
//        Exact unless a product is NaN (a NaN makes the chain forget what came before): dist_merge.hip has the detector
//        and the sequential redo that go with it.
//   min, "around" form (round 5; vc.n != 0) - both sides in ONE launch: the matrix is written in the row order of the whole
//        shard, [columns that precede | ONE virtual entry | columns that follow], the virtual entry (column id vc.lo + output
//        row, weight 1, only in rows whose output pair is not the empty row's) standing for everything (C, E)[output row]
//        already cover: its "dense row" is that row of C (dense_row above), so the old value goes through the row's own
//        chain / tree / partial rows at its place in the row - every tie rule is the row's own, nothing is merged by key -
//        and the commit only has to write the result and, where the virtual entry won, keep the arg the output held.
//        Every reader of C[row] belongs to row `row` and has consumed it before the row's commit (one wave; or the row's unit
//        waves, whose partial rows the commit folds), so the launch works in place.  Real columns >= vc.lo + vc.n are
//        B rows shifted by vc.n (the ids of a sorted shard row stay sorted: the plan can cut by column slice).
struct AccArg {
  const int *rowmap;  // output row of every row of A (nullptr = identity)
  int col_off;        // added to this product's arg column ids (halo slot -> extended id)
  int nl, h_lo;       // max: extended-id layout: local columns [0, nl), h_lo of the halo slots precede them; min: see above
  Epi epi;            // plain (non-accumulating) sum / mean only: bias / row scale / relu at the row-end store
  VirtCols vc;        // min, "around" form
};
template <int OP>
constexpr bool epi_op() { return OP == DGS_SUM || OP == DGS_MEAN; }
__device__ __forceinline__ int acc_key(int e, int nl, int h_lo) { return e < nl ? h_lo + e : (e - nl < h_lo ? e - nl : e); }

template <int V, int OP, bool HIDDEN>
__device__ __forceinline__ void acc_commit(float *__restrict__ C, int *__restrict__ E, int64_t orow, int N, int f0,
                                           const float (&acc)[V], const int (&ei)[V], const AccArg &aa) {
  float *cp = C + orow * N + f0;
  float old[V];
  load_vec<V>(cp, old);
  if constexpr (OP == DGS_MAX) {
    int *ep = E + orow * N + f0;
    int eo[V];
    load_vec<V>(ep, eo);
    // Branch-free on purpose, results in fresh arrays: hipcc 7.2 miscompiled the short-circuit form of this merge for
    // V = 4 (a 64-bit register-pair move clobbered the kept value of the neighbouring feature).
    float cv[V];
    int ev[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int en = ei[v] >= 0 ? ei[v] + aa.col_off : -1;
      const int kn = acc_key(en, aa.nl, aa.h_lo), ko = acc_key(eo[v], aa.nl, aa.h_lo);
      const int better = (int)(eo[v] < 0) | (int)(old[v] < acc[v]) | ((int)(old[v] == acc[v]) & (int)(kn < ko));
      const bool take = ((int)(en >= 0) & better) != 0;
      cv[v] = take ? acc[v] : old[v];
      ev[v] = take ? en : eo[v];
    }
    if constexpr (HIDDEN) {
      store_vec_hidden<V>(ep, ev);
      store_vec_hidden<V>(cp, cv);
    } else {
      store_vec_stream<V>(ep, ev);
      store_vec_stream<V>(cp, cv);
    }
  } else if constexpr (OP == DGS_MIN) {
    int *ep = E + orow * N + f0;
    int eo[V];
    load_vec<V>(ep, eo);
    const bool first = aa.h_lo != 0;  // this product's columns precede the ones (old, eo) cover
    const bool around = aa.vc.n != 0;  // the old pair went through the row as its virtual entry: (acc, ei) is the whole result
    float cv[V];
    int ev[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
      // (around: ids below vc.lo are the slots that precede, ids from vc.lo + vc.n on the slots that follow, shifted by vc.n)
      const int es = (around & (ei[v] >= aa.vc.lo)) ? ei[v] - aa.vc.n : ei[v];
      const int en = ei[v] >= 0 ? es + aa.col_off : -1;
      // (ei < 0: nothing improved on the identity, the virtual entry included - a NaN that ended the old pair's own chain does not, and
      // neither did anything behind it: the old arg stands)
      const bool won_virt = around & (((unsigned)(ei[v] - aa.vc.lo) < (unsigned)aa.vc.n) | (ei[v] < 0));
      const float a = first ? acc[v] : old[v], b = first ? old[v] : acc[v];  // a comes first in the row
      const int ea = first ? en : eo[v], eb = first ? eo[v] : en;
      const bool old_empty = (eo[v] < 0) & (old[v] != reduce_init<DGS_MIN>());
      // algorithm 0's step with res = a, t = b (branch-free, fresh arrays: see the max case)
      const float mv = (a < b) ? a : b;
      const int me = (a > b) ? eb : ea;
      cv[v] = (old_empty | around) ? acc[v] : mv;
      ev[v] = won_virt ? eo[v] : ((old_empty | around) ? en : me);
    }
    if constexpr (HIDDEN) {
      store_vec_hidden<V>(ep, ev);
      store_vec_hidden<V>(cp, cv);
    } else {
      store_vec_stream<V>(ep, ev);
      store_vec_stream<V>(cp, cv);
    }
  } else {
    float cv[V];
#pragma unroll
    for (int v = 0; v < V; v++) cv[v] = acc[v] + old[v];
    if constexpr (HIDDEN) store_vec_hidden<V>(cp, cv);
    else store_vec_stream<V>(cp, cv);
  }
}

// ACC (sum only): C[out row] += result instead of C[row] = result, out row = rowmap[row] when a map is given (the
// halo product of dgsparse.dist adds into the rows that have remote entries); rows without entries are left alone.
// STRICT (spmm_strict.h; sum / mean only): 0 = default; 1 = every row one sequential fmaf chain; 2 = the same without
// contraction.  Here it only changes the arithmetic of the (already sequential) short rows and, in the single-launch
// kernel, sends the long rows through strict_unit instead of the wave-cooperative tree.  3 = the default arithmetic, the single-launch
// kernel's rows above `thub` nnz skipped and reported in `hubmask` (two words per wave; spmm_small_hub chains them).
template <int G, int V, int OP, bool HAS_VAL, bool INLINE, bool ACC = false, int STRICT = 0>
__device__ __forceinline__ void spmm_rows_body(int bid, int rpw, RowsLds &lds, int M, int N,
                                               const int *__restrict__ rowptr,
                                               const int *__restrict__ col, const float *__restrict__ val,
                                               const float *__restrict__ B, float *__restrict__ C,
                                               int *__restrict__ E, const AccArg aa = AccArg{},
                                               float *strict_xb = nullptr, const int thub = INT_MAX,
                                               unsigned *hubmask = nullptr) {
  static_assert(!ACC || OP == DGS_SUM || OP == DGS_MAX || OP == DGS_MIN, "accumulation exists for sum, max and min");
  static_assert(STRICT == 0 || ((OP == DGS_SUM || OP == DGS_MEAN) && !ACC), "strict order exists for plain sum and mean");
  const int *rowmap = aa.rowmap;
  constexpr int NG = kWave / G;
  constexpr bool ARG = (OP == DGS_MAX || OP == DGS_MIN);
  constexpr bool VIRT = ACC && OP == DGS_MIN;  // the only instantiations that know virtual columns (AccArg, "around" form)
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int g = lane / G, l = lane % G;
  const int r0 = (bid * (kBlock / kWave) + wave) * rpw;  // rpw <= 64 rows per wave (fewer on small inputs)
  if (r0 >= M) return;  // wave-uniform
  [[maybe_unused]] const int trace_id = bid * (kBlock / kWave) + wave;
  DGS_TS(0);
  int2 *tile = lds.tile[wave];
  int4 *rows = lds.rows[wave];
  const int nrows = min(rpw, M - r0);
  const int f0 = (blockIdx.y * G + l) * V;
  const bool fl = f0 < N;

  int s_i = 0, e_i = 0;
  if (lane < nrows) {
    s_i = rowptr[r0 + lane];
    e_i = rowptr[r0 + lane + 1];
  }
  const int len_i = e_i - s_i;
  const bool long_i = len_i > kT1;   // not streamed: medium (whole wave, below) or huge (unit table)
  const bool huge_i = !INLINE && len_i > kT2;  // INLINE (small inputs, single launch): no unit table at all
  const bool live_i = lane < nrows && len_i > 0 && !long_i;  // non-empty short row: produces output in the stream
  {
    // index of the next live row after this lane's row (64 = none)
    const unsigned long long livemask = __ballot(live_i);
    const unsigned long long above = (lane >= 63) ? 0ull : (livemask >> (lane + 1));
    const int nxt = above ? (lane + 1 + (__ffsll((long long)above) - 1)) : kRowsPerWave;
    int orow_i = 0;
    if constexpr (ACC) orow_i = (lane < nrows) ? (rowmap ? rowmap[r0 + lane] : r0 + lane) : 0;
    rows[lane] = make_int4(s_i, e_i, nxt, orow_i);
    // empty rows: 0 / E = -1 (spmm_cuda.cuh:49-51); NG rows per pass, one per group
    unsigned long long em = ACC ? 0ull : __ballot(lane < nrows && len_i == 0);
    while (em) {
      int r = -1;
      unsigned long long t = em;
      for (int k = 0; k <= g && t; k++) {  // g-th set bit
        r = __ffsll((long long)t) - 1;
        t &= t - 1;
        if (k < g) r = -1;
      }
      if (r >= 0 && fl) {
        float z[V];
        int m1[V];
#pragma unroll
        for (int v = 0; v < V; v++) {
          z[v] = 0.0f;
          m1[v] = -1;
        }
        if constexpr (epi_op<OP>()) epi_apply<V>(z, r0 + r, f0, aa.epi);
        store_vec_stream<V>(C + (int64_t)(r0 + r) * N + f0, z);
        if constexpr (ARG) store_vec_stream<V>(E + (int64_t)(r0 + r) * N + f0, m1);
      }
      for (int k = 0; k < NG && em; k++) em &= em - 1;  // drop the NG rows just written
    }
  }

  DGS_TS(1);  // rowptr arrived (ballots above consumed it), row table in LDS, empty rows written
  int a = 0;
  while (a < nrows) {
    const int s_a = __shfl(s_i, a, 64);
    // first row >= a that cannot join the batch: long, or it would overflow the LDS tile, or past the end
    const unsigned long long brk = __ballot(lane >= a && (long_i || (e_i - s_a) > kCap || lane >= nrows));
    const int b = brk ? (__ffsll((long long)brk) - 1) : kRowsPerWave;
    if (b == a) {  // row a itself is long: skipped here
      a++;
      continue;
    }
    const int e_b = __shfl(e_i, b - 1, 64);
    const int cnt = e_b - s_a;
    if (cnt == 0) {  // only empty rows in this run
      a = b;
      continue;
    }
    __builtin_amdgcn_wave_barrier();
    // (one pass per 64 entries; issuing all passes' loads before the first LDS store was tried after the per-wave
    // timeline showed 24 % / 61 % of a row wave's life here (arxiv-shaped / headline graph): no change in that share - the
    // wait is the queueing delay of a streaming load behind the CU's gathers, not a chain - and the 16 extra live
    // registers cost the max kernel 4 %)
    for (int t = lane; t < cnt; t += kWave) {
      const int c = ld_stream(col + s_a + t);
      const float w = HAS_VAL ? ld_stream(val + s_a + t) : 1.0f;
      tile[t] = make_int2(c, __float_as_int(w));
    }
    __builtin_amdgcn_wave_barrier();
    DGS_TS(2);  // (col,val) tile staged
    // row-end flag = sign bit of the column id of each live row's last nnz (column ids are < 2^31)
    if (live_i && lane >= a && lane < b) tile[e_i - 1 - s_a].x |= (int)0x80000000;
    __builtin_amdgcn_wave_barrier();

    // piece of group g: rows [ra, rb) where boundary(k) = first row r in [a,b] with start_r - s_a >= k*cnt/NG
    int ra, rb;
    if constexpr (NG <= 16) {
      // every lane still holds its row's start: boundary k is the first set bit of one ballot (no LDS round trips)
      ra = a;
      rb = b;
      const bool in_run = lane >= a && lane < b;
      for (int k = 1; k < NG; k++) {
        const int tgt = (int)(((long long)k * cnt) / NG);
        const unsigned long long m = __ballot(in_run && (s_i - s_a) >= tgt);
        const int bk = m ? (__ffsll((long long)m) - 1) : b;
        if (g == k) ra = bk;
        if (g + 1 == k) rb = bk;
      }
    } else {
      const int tgt0 = (int)(((long long)g * cnt) / NG), tgt1 = (int)(((long long)(g + 1) * cnt) / NG);
      int lo = a, hi = b;  // first r in [a,b] with rows[r].x - s_a >= tgt0   (rows[b].x >= e_b by CSR monotonicity)
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const int sm = (mid < b) ? rows[mid].x : e_b;
        if (sm - s_a < tgt0) lo = mid + 1; else hi = mid;
      }
      ra = lo;
      lo = ra;
      hi = b;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const int sm = (mid < b) ? rows[mid].x : e_b;
        if (sm - s_a < tgt1) lo = mid + 1; else hi = mid;
      }
      rb = (g == NG - 1) ? b : lo;
    }
    DGS_TS(3);  // piece boundaries found
    if (ra < rb) {
      const int ps = rows[ra].x - s_a;
      const int pe = ((rb < b) ? rows[rb].x : e_b) - s_a;
      // first live row of the piece
      int cur = ra;
      {
        const int4 q = rows[ra];
        if (!(q.y > q.x)) cur = q.z;
      }
      float acc[V];
      int ei[V];
#pragma unroll
      for (int v = 0; v < V; v++) {
        acc[v] = reduce_init<OP>();
        ei[v] = -1;
      }
      // Rolling window of kU1 gathers: slot i always holds nnz (p+i); after it is consumed the slot is refilled
      // with nnz (p+i+kU1).  Loads are unconditional (index clamped to the last nnz of the piece, feature lanes
      // beyond N read feature 0) so the compiler emits counted s_waitcnt vmcnt(kU1-1) instead of draining.
      const float *Bl = B + (fl ? f0 : 0);
      VirtCols vcl = aa.vc;  // (the lane's feature offset folded into the base, like Bl)
      if constexpr (VIRT) vcl.C = aa.vc.C + (fl ? f0 : 0);
      const int last = pe - 1;
      int2 cv[kU1];
      float x[kU1][V];
      int mk[kU1][V];
      const int *El = OP == kOpMaskSum ? E + (fl ? f0 : 0) : nullptr;
#pragma unroll
      for (int u = 0; u < kU1; u++) {
        cv[u] = tile[min(ps + u, last)];
        load_vec_gather<V>(dense_row<VIRT>(Bl, cv[u].x & 0x7fffffff, N, vcl), x[u]);
        if constexpr (OP == kOpMaskSum) load_vec<V>(El + (int64_t)(cv[u].x & 0x7fffffff) * N, mk[u]);
        // keep the fill in slot order: hipcc otherwise issues slot 0 LAST, and the loop's first wait - merged over the
        // entry edge and the back edge - becomes vmcnt(1), a drain of the whole window once per kU1 gathers
        __builtin_amdgcn_sched_barrier(0);
      }
      for (int p = ps; p < pe; p += kU1) {
#pragma unroll
        for (int u = 0; u < kU1; u++) {
          const int2 cvu = cv[u];
          if (p + u < pe) {
            const int c = cvu.x & 0x7fffffff;
            const float w = __int_as_float(cvu.y);
#pragma unroll
            for (int v = 0; v < V; v++) {
              if constexpr (OP == kOpMaskSum) {
                if (mk[u][v] == r0 + cur) acc[v] = __builtin_fmaf(w, x[u][v], acc[v]);
              } else {
                reduce_step<OP, STRICT != 2>(acc[v], ei[v], w, x[u][v], c);
              }
            }
            if (cvu.x < 0) {  // last nnz of row `cur` (group-uniform)
              const int4 q = rows[cur];
              if constexpr (OP == DGS_MEAN) {
                const float d = (float)(q.y - q.x);
#pragma unroll
                for (int v = 0; v < V; v++) acc[v] /= d;
              }
              if (fl) {
                if constexpr (ACC) {
                  acc_commit<V, OP, true>(C, E, q.w, N, f0, acc, ei, aa);
                } else {
                  if constexpr (epi_op<OP>()) epi_apply<V>(acc, r0 + cur, f0, aa.epi);
                  store_vec_hidden<V>(C + (int64_t)(r0 + cur) * N + f0, acc);
                  if constexpr (ARG) store_vec_hidden<V>(E + (int64_t)(r0 + cur) * N + f0, ei);
                }
              }
#pragma unroll
              for (int v = 0; v < V; v++) {
                acc[v] = reduce_init<OP>();
                ei[v] = -1;
              }
              cur = q.z;
            }
          }
          // refill the slot just consumed (same registers: no copies, so the waits stay counted)
          // (reading the tile entry one step ahead, so that its LDS latency runs under the wait for the oldest gather, was
          // built and measured late in round 3: no change anywhere - arxiv-shaped 48.0 us, headline 0.390 ms - and dropped)
          cv[u] = tile[min(p + u + kU1, last)];
          load_vec_gather<V>(dense_row<VIRT>(Bl, cv[u].x & 0x7fffffff, N, vcl), x[u]);
          if constexpr (OP == kOpMaskSum) load_vec<V>(El + (int64_t)(cv[u].x & 0x7fffffff) * N, mk[u]);
        }
      }
    }
    DGS_TS(4);  // gather loop of the batch done
    a = b;
  }
  DGS_TS(5);

  // medium rows (T1 < len <= T2): the whole wave reduces one row at a time, result written directly
  unsigned long long med = __ballot(long_i && !huge_i);
  while (med) {
    const int r = __ffsll((long long)med) - 1;
    med &= med - 1;
    const int rs = __shfl(s_i, r, 64), re = __shfl(e_i, r, 64);
    if constexpr (STRICT == 1 || STRICT == 2) {
      strict_unit<V, G, OP == DGS_MEAN, HAS_VAL, STRICT != 2>(r0 + r, rs, re - rs, blockIdx.y * G * V, 0, lane, N, col, val, B,
                                                             C, strict_xb);
      continue;
    }
    if constexpr (STRICT == 3) {
      if (re - rs > thub) {  // wave-uniform: left to the workgroup (spmm_small_hub), bit = row inside this wave's range
        if (lane == 0) hubmask[wave * 2 + (r >> 5)] = hubmask[wave * 2 + (r >> 5)] | (1u << (r & 31));
        continue;
      }
    }
    float acc[V];
    int ei[V], ep[V], el[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
      acc[v] = reduce_init<OP>();
      ei[v] = -1;
      ep[v] = INT_MAX;
      el[v] = -1;
    }
    float nf[V] = {};
    coop_accumulate<G, V, OP, HAS_VAL, VIRT>(rs, re, lane, g, f0, fl, N, col, val, B, E, r0 + r, tile, acc, ei, ep, el, nf, aa.vc);
    cross_group_reduce<G, V, OP>(acc, ei, ep, el);
    if constexpr (OP == DGS_MIN) {
      const unsigned nm = nan_flags<G, V>(nf);
      if (nm && g == 0 && fl) seq_redo<V, OP, VIRT>(nm, rs, re, N, f0, col, HAS_VAL ? val : nullptr, B, acc, ei, aa.vc);
    }
    if (g == 0 && fl) {
      if constexpr (OP == DGS_MEAN) {
        const float dg = (float)(re - rs);
#pragma unroll
        for (int v = 0; v < V; v++) acc[v] /= dg;
      }
      if constexpr (ACC) {
        acc_commit<V, OP, false>(C, E, rows[r].w, N, f0, acc, ei, aa);
      } else {
        if constexpr (epi_op<OP>()) epi_apply<V>(acc, r0 + r, f0, aa.epi);
        store_vec_stream<V>(C + (int64_t)(r0 + r) * N + f0, acc);
        if constexpr (ARG) store_vec_stream<V>(E + (int64_t)(r0 + r) * N + f0, ei);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// Fold of ONE multi-unit row by one wave: the row's partial rows in unit order (groups take interleaved units, UP independent
// partial loads in flight per lane, then the fixed cross-group tree), MIN's NaN redo, mean, epilogue, store.  Two callers: the
// combine kernel (K3: one wave per entry of the long-row table, after the fused launch) and - round 5, COH = true - the unit wave
// that completed the row inside the fused launch (spmm_units_body: last arriver), which reads the partial rows other workgroups
// - other XCDs - wrote moments ago: those loads are agent-scope (sc1: past the XCD's own L2), like the stores that wrote them.
#ifndef DGS_COMBINE_UP
#define DGS_COMBINE_UP 8  // partial rows in flight per lane: 4 -> 8 takes the fold of a 400-unit hub row from 25 to 13 dependent rounds (combine 13.6 -> ~8 us on the headline graph, 8.7 -> 6.5 us arxiv-shaped); 16 adds little
#endif
#ifndef DGS_COMBINE_UP_ARG
#define DGS_COMBINE_UP_ARG 4  // max / min carry (value, arg) per partial row: 8 in flight cost 134 VGPRs = 3 waves per SIMD
#endif
// Agent-coherent accesses to the partial rows (COH: the in-kernel fold).  16-byte lanes go through ONE buffer instruction with the
// sc1 bit per lane (`buffer_store_dwordx4 ... sc1`: write-through; `buffer_load_dwordx4 ... sc1`: past the CU's L1) - a relaxed
// agent-scope __hip_atomic_store / _load lowers to an sc1 access only up to 8 bytes, and every scalar sc1 store is a fabric write
// of its own (MI355X guide, "Workgroup dispatch ... inter-workgroup visibility": dword ~6x the dwordx4 time per byte; its R1 form:
// 16-byte sc1 stores -> s_waitcnt vmcnt(0) -> relaxed agent-scope counter; reader: returned atomic -> sc1 loads).  The compiler
// counts buffer loads like any other load, so the fold's "every load issued, one wait" structure is unchanged.  The descriptor
// covers the whole partial-row region (wave-uniform: kernel arguments only); the launcher only folds in the kernel when that
// region is below 2^31 bytes (fold_fits), so a 32-bit byte offset reaches every slot.  Scalar lanes keep the 4-byte atomics.
typedef unsigned int dgs_u4 __attribute__((ext_vector_type(4)));
constexpr int kAuxSc1 = 16;  // cache-policy operand of the raw buffer builtins on gfx942 / gfx950: bit 4 = sc1
struct CohBuf {
  __amdgpu_buffer_rsrc_t rs;
};
__device__ __forceinline__ CohBuf coh_buf(const void *base, unsigned bytes) {
  return CohBuf{__builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (int)bytes, 0x00020000)};
}
template <int V, bool COH, typename T>
__device__ __forceinline__ void load_part(const T *base, const int64_t idx, const CohBuf &cb, T (&o)[V]) {
  static_assert(sizeof(T) == 4, "partial rows are float / int32");
  if constexpr (COH && V == 4) {
    const dgs_u4 u = __builtin_amdgcn_raw_buffer_load_b128(cb.rs, (int)(idx * 4), 0, kAuxSc1);
    __builtin_memcpy(o, &u, 16);
  } else if constexpr (COH) {
#pragma unroll
    for (int v = 0; v < V; v++) o[v] = __hip_atomic_load(base + idx + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  } else {
    load_vec<V>(base + idx, o);
  }
}
template <int V, typename T>
__device__ __forceinline__ void store_part_coherent(T *base, const int64_t idx, const CohBuf &cb, const T (&o)[V]) {
  static_assert(sizeof(T) == 4, "partial rows are float / int32");
  if constexpr (V == 4) {
    dgs_u4 u;
    __builtin_memcpy(&u, o, 16);
    __builtin_amdgcn_raw_buffer_store_b128(u, cb.rs, (int)(idx * 4), 0, kAuxSc1);
  } else {
#pragma unroll
    for (int v = 0; v < V; v++) __hip_atomic_store(base + idx + v, o[v], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}
template <int G, int V, int OP, bool ACC, bool COH>
__device__ __forceinline__ void fold_row(const int4 d, const int lane, const int N, const int *__restrict__ rowptr,
                                         const int *__restrict__ col, const float *__restrict__ val,
                                         const float *__restrict__ B, float *__restrict__ C, int *__restrict__ E,
                                         const float *__restrict__ part, const int *__restrict__ parte, const AccArg &aa,
                                         const unsigned part_bytes = 0, const int pstride = 0) {
  constexpr int NG = kWave / G;
  const int ps = COH ? pstride : N;  // floats between two partial rows (COH: whole lines per slot, fold_stride)
  constexpr bool ARG = (OP == DGS_MAX || OP == DGS_MIN);
  const CohBuf cbp = coh_buf(part, COH ? part_bytes : 0), cbe = coh_buf(ARG ? (const void *)parte : (const void *)part, COH ? part_bytes : 0);
  // max: a partial row that never improved on the identity carries the identity as its value, so the fold needs values and
  // positions only; the arg id of each element's winner is fetched once at the end (half the loads, 8 rows in flight again)
  constexpr bool LATE_ARG = (OP == DGS_MAX);
  constexpr int UP = (ARG && !LATE_ARG) ? DGS_COMBINE_UP_ARG : DGS_COMBINE_UP;
  const int g = lane / G, l = lane % G;
  const int f0 = (blockIdx.y * G + l) * V;
  const bool fl = f0 < N;
  float acc[V];
  int ei[V], ep[V], el[V];
  unsigned nm = 0;  // MIN: elements whose partials met a NaN product
#pragma unroll
  for (int v = 0; v < V; v++) {
    acc[v] = reduce_init<OP>();
    ei[v] = -1;
    ep[v] = INT_MAX;
    el[v] = -1;
  }
  for (int k = g; k < d.z; k += NG * UP) {
    float x[UP][V];
    int xe[UP][V];
    // every load is issued, with its index clamped into the row's slots: conditional loads end up in basic blocks of their
    // own, and hipcc's waitcnt pass then puts a vmcnt(1) in front of each - 8 dependent latencies per round instead of
    // one (ISA read, late round 3: combine of max 54.8 us for 10.4 us of sum on the headline graph)
#pragma unroll
    for (int q = 0; q < UP; q++) {
      const int64_t slot = (int64_t)(d.y + min(k + q * NG, d.z - 1)) * ps + (fl ? f0 : 0);
      load_part<V, COH>(part, slot, cbp, x[q]);
      if constexpr (ARG && !LATE_ARG) load_part<V, COH>(parte, slot, cbe, xe[q]);
    }
    // branch-free folds (selects on fresh values): the merges of one round are 32 short data-dependent branches otherwise
#pragma unroll
    for (int q = 0; q < UP; q++) {
      const int pos = k + q * NG;
      const bool valid = (pos < d.z) & fl;
#pragma unroll
      for (int v = 0; v < V; v++) {
        if constexpr (OP == DGS_MIN) {
          // units arrive in increasing k inside a group: a strictly smaller partial takes everything, an equal one
          // only refreshes the value (later operand wins ties in the MIN macro); E=-1 partials never improved
          const bool nanp = valid & (xe[q][v] == kNanMark);
          const bool live = valid & (xe[q][v] != kNanMark) & (xe[q][v] != -1);
          const bool lt = live & (acc[v] > x[q][v]);
          const bool le = lt | (live & (acc[v] == x[q][v]));
          nm |= nanp ? (1u << v) : 0u;
          acc[v] = le ? x[q][v] : acc[v];
          ei[v] = lt ? xe[q][v] : ei[v];
          ep[v] = lt ? pos : ep[v];
          el[v] = le ? pos : el[v];
        } else if constexpr (ARG) {
          // a partial that never improved on the identity (E = -1) holds the identity itself: it can take the position of
          // another such partial, never that of a real one, and the arg id fetched for it at the end is its -1
          const bool take = valid & arg_better<OP>(acc[v], ep[v], x[q][v], pos);
          acc[v] = take ? x[q][v] : acc[v];
          ep[v] = take ? pos : ep[v];
        } else {
          if (valid) acc[v] += x[q][v];
        }
      }
    }
  }
  cross_group_reduce<G, V, OP>(acc, ei, ep, el);
  if constexpr (LATE_ARG) {
    if (g == 0 && fl) {
#pragma unroll
      for (int v = 0; v < V; v++) {
        if (ep[v] != INT_MAX) {
          const int *q = parte + (int64_t)(d.y + ep[v]) * ps + f0 + v;
          ei[v] = COH ? __hip_atomic_load(q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *q;
        } else {
          ei[v] = -1;
        }
      }
    }
  }
  if constexpr (OP == DGS_MIN) {
#pragma unroll
    for (int dd = G; dd < 64; dd <<= 1) nm |= (unsigned)__shfl_xor((int)nm, dd, 64);
    if (nm && g == 0 && fl) seq_redo<V, OP, ACC && OP == DGS_MIN>(nm, rowptr[d.x], rowptr[d.x + 1], N, f0, col, val, B, acc, ei, aa.vc);
  }
  if (g == 0 && fl) {
    if constexpr (OP == DGS_MEAN) {
      const float dg = (float)(rowptr[d.x + 1] - rowptr[d.x]);
#pragma unroll
      for (int v = 0; v < V; v++) acc[v] /= dg;
    }
    if constexpr (ACC) {
      acc_commit<V, OP, false>(C, E, aa.rowmap ? aa.rowmap[d.x] : d.x, N, f0, acc, ei, aa);
    } else {
      if constexpr (epi_op<OP>()) epi_apply<V>(acc, d.x, f0, aa.epi);
      store_vec_stream<V>(C + (int64_t)d.x * N + f0, acc);
      if constexpr (ARG) store_vec_stream<V>(E + (int64_t)d.x * N + f0, ei);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// K2: one wave per unit (<= ch nnz of a long row).
template <int G, int V, int OP, bool HAS_VAL, bool ACC = false, bool FOLD = false>
__device__ __forceinline__ void spmm_units_body(int bid, int nblocks, RowsLds &lds, int N,
                                                const int *__restrict__ rowptr, const int *__restrict__ col,
                                                const float *__restrict__ val, const float *__restrict__ B,
                                                float *__restrict__ C, int *__restrict__ E, const UnitTab &ut,
                                                float *__restrict__ part, int *__restrict__ parte,
                                                const AccArg aa = AccArg{}) {
  constexpr bool ARG = (OP == DGS_MAX || OP == DGS_MIN);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int g = lane / G, l = lane % G;
  int2 *tile = lds.tile[wave];
  const int f0 = (blockIdx.y * G + l) * V;
  const bool fl = f0 < N;
  const int n_units = *ut.n_units;
  // XCD-aware unit mapping (speed hint only): block b runs on XCD b % 8 (observed), so the unit blocks of one XCD walk
  // one contiguous share of the table: a few runs of neighbouring rows (spmm_classify), or - with a plan - the units of
  // ONE COLUMN SLICE in column order, so that an XCD's L2 only ever sees an eighth of the dense operand.
  int u, uend, wstride;
#if DGS_XCD_REMAP
  if ((nblocks & 7) == 0) {
    const int x = bid & 7, wx = (nblocks >> 3) * (kBlock / kWave);
    const int lo = ut.xcd_start ? ut.xcd_start[x] : (int)(((long long)n_units * x) >> 3);
    uend = ut.xcd_end ? ut.xcd_end[x] : (ut.xcd_start ? ut.xcd_start[x + 1] : (int)(((long long)n_units * (x + 1)) >> 3));
    u = lo + (bid >> 3) * (kBlock / kWave) + wave;
    wstride = wx;
  } else
#endif
  {
    u = bid * (kBlock / kWave) + wave;
    uend = n_units;
    wstride = nblocks * (kBlock / kWave);
  }
  // In-kernel fold (ut.arrive != nullptr): a unit's partial row is written with agent-scope stores, and ONE unit later - when the
  // wave has waited for that unit's gathers anyway, so the stores are long complete and the wait below is free - the wave counts
  // the unit in on its row's arrival counter; whoever brings the count to the row's number of units folds the row right here
  // (fold_row: fixed unit order, so the result does not depend on who that is).  Ordering: stores performed at agent scope
  // (s_waitcnt vmcnt(0)) -> atomic add on the counter -> the last arriver's loads, issued after its own add has returned (and
  // been looked at: one more unit later, see count_in / settle).
  // FOLD is a COMPILE-TIME choice (round 6): the ticket state and the fold's eight-deep window of partial rows cost the max / min
  // instantiations 10 - 35 spilled VGPRs (`<16, 4, MAX>` 0 -> 13, `<16, 4, MIN>` 10 -> 41, `<8, 4, MIN>` 55 -> 90 against round 3's
  // code objects; the masked sum 40 -> 61) when it was a run-time branch inside the one instantiation every call
  // took.  The default launch (fold off, launch_fused) is now an instantiation without any of it - register for register the
  // hardware-verified round-3 unit body plus the hub role - and DGS_FOLD=1 | 2 selects the FOLD = true twin (never built for the
  // masked sum: its unit body already carries the gradient AND the arg-id gather windows).
  constexpr bool folding = FOLD;
  const CohBuf cbp = coh_buf(part, folding ? ut.part_bytes : 0), cbe = coh_buf(ARG ? (void *)parte : (void *)part, folding ? ut.part_bytes : 0);
  int pend = -1;  // long-row index of the partial row this wave wrote last and has not counted in yet
  // ... and one step further down the pipeline: the row whose counter this wave has incremented WITHOUT having looked at the
  // returned count yet.  A returning device-scope atomic takes ~0.25 us on an idle chip and ~1.1 us under streaming load (MI355X
  // guide, hand-off price list: "dequeue"); waited for on the spot, that is 5 - 10 % of a unit's life with the wave issuing
  // nothing.  So the count is read ONE UNIT LATER (settle), when it has long returned - like the partial-row stores, whose drain
  // in front of the atomic is free because they are a unit old.  At most one ticket per wave is in flight.
  int tick_row = -1, tick_old = 0;
  auto count_in = [&](int li) {
    drain_vmem();  // s_waitcnt vmcnt(0), as inline asm: this wave's partial-row stores have been performed (written through)
    // (one counter per long row AND feature tile: the tiles of a launch fold independently)
    if (lane == 0)
      tick_old = __hip_atomic_fetch_add(ut.arrive + (int64_t)li * gridDim.y + blockIdx.y, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    tick_row = li;
  };
  auto settle = [&]() {
    if (tick_row < 0) return;  // wave-uniform
    const int old = __shfl(tick_old, 0, 64);
    const int4 lr = ut.longrows[tick_row];  // {row, first partial slot, units in the row, -}
    tick_row = -1;
    if (old == lr.z - 1) {  // this wave brought the count to the row's number of units: every partial row has been written through
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      fold_row<G, V, OP, ACC, true>(lr, lane, N, rowptr, col, HAS_VAL ? val : nullptr, B, C, E, part, parte, aa, ut.part_bytes, ut.pstride);
    }
  };
  for (; u < uend; u += wstride) {
    const int4 d = ut.units[u];  // {row, first nnz, nnz in the unit, partial slot | -1}
    const int p0 = d.y, p1 = d.y + d.z;
    const bool whole = d.w < 0;
    float acc[V];
    int ei[V], ep[V], el[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
      acc[v] = reduce_init<OP>();
      ei[v] = -1;
      ep[v] = INT_MAX;
      el[v] = -1;
    }
    float nf[V] = {};
    coop_accumulate<G, V, OP, HAS_VAL, ACC && OP == DGS_MIN>(p0, p1, lane, g, f0, fl, N, col, val, B, E, d.x, tile, acc, ei, ep, el, nf, aa.vc);
    cross_group_reduce<G, V, OP>(acc, ei, ep, el);
    if constexpr (OP == DGS_MIN) {
      const unsigned nm = nan_flags<G, V>(nf);
      if (nm && g == 0 && fl) {
        if (whole) {
          seq_redo<V, OP, ACC && OP == DGS_MIN>(nm, p0, p1, N, f0, col, HAS_VAL ? val : nullptr, B, acc, ei, aa.vc);
        } else {  // tell the combine kernel to redo these elements of the row
#pragma unroll
          for (int v = 0; v < V; v++)
            if (nm >> v & 1) ei[v] = kNanMark;
        }
      }
    }
    if (folding) {
      settle();         // the ticket drawn one unit ago: its count has long returned
      if (pend >= 0) {  // the previous partial row of this wave: its stores are a whole unit old, the drain is free
        count_in(pend);
        pend = -1;
      }
    }
    if (g == 0 && fl) {
      if (whole) {  // the whole row was this unit: final result
        if constexpr (OP == DGS_MEAN) {
          const float dg = (float)d.z;
#pragma unroll
          for (int v = 0; v < V; v++) acc[v] /= dg;
        }
        if constexpr (ACC) {
          acc_commit<V, OP, false>(C, E, aa.rowmap ? aa.rowmap[d.x] : d.x, N, f0, acc, ei, aa);
        } else {
          if constexpr (epi_op<OP>()) epi_apply<V>(acc, d.x, f0, aa.epi);
          store_vec_stream<V>(C + (int64_t)d.x * N + f0, acc);
          if constexpr (ARG) store_vec_stream<V>(E + (int64_t)d.x * N + f0, ei);
        }
      } else {
        const int64_t slot = (int64_t)d.w * (FOLD ? ut.pstride : N) + f0;
        if (folding) {
          store_part_coherent<V>(part, slot, cbp, acc);
          if constexpr (ARG) store_part_coherent<V>(parte, slot, cbe, ei);
        } else {
          store_vec<V>(part + slot, acc);
          if constexpr (ARG) store_vec<V>(parte + slot, ei);
        }
      }
    }
    if (folding && !whole) pend = ut.slot_long[d.w];
  }
  if (folding) {  // drain the pipeline: the ticket in flight, then the last partial row
    settle();
    if (pend >= 0) count_in(pend);
    settle();
  }
}

// ---------------------------------------------------------------------------------------------------------
// Waves per SIMD the fused kernel is compiled for.  The kernel hides DRAM latency with waves, not with a deep per-wave
// pipeline: max went 0.650 -> 0.523 ms on the headline graph when 106 VGPRs (4 waves) became 96 (5 waves, 6 spilled).
#ifndef DGS_WAVES_SUM
#define DGS_WAVES_SUM 5
#endif
#ifndef DGS_WAVES_ARG
#define DGS_WAVES_ARG 5
#endif
// (The opt-in fold twins of min and mean hold the ticket state as well: one wave less, instead of 12 - 42 spilled registers.)
constexpr int fused_waves_per_simd(int op, bool fold) {
  return ((op == DGS_MAX || op == DGS_MIN) ? DGS_WAVES_ARG : DGS_WAVES_SUM) - (fold && (op == DGS_MIN || op == DGS_MEAN) ? 1 : 0);
}

// Fused launch: blocks [0, nbu) walk the unit table of the huge rows (persistent, strided), the remaining blocks
// each own 4 x 64 consecutive rows.  Unit blocks come first so that the longest-running work starts first; the
// two kinds of work share the CUs, so the fabric-bound unit gathers overlap the row kernel's latency phases.
// HUB (sum / mean, 16-byte lanes, tiles of >= 16 floats): the first nbh blocks chain the hub rows (spmm_hub_body: every row
// longer than the hub threshold one sequential fmaf chain per feature, like the rows up to T1 - the rows in between keep the
// fixed tree); they come first in the grid because a 50 k-nnz chain is the longest job of the launch.
template <int OP, int V, int G, bool ACC>
constexpr bool hub_ok() { return DGS_HUB_COOP_V2 && (OP == DGS_SUM || OP == DGS_MEAN) && !ACC && strict_coop(G, V); }
struct HubLds {
  alignas(16) float f[kHubBlockFloats];
};
template <bool HUB>
struct FusedLds {
  RowsLds r;
};
template <>
struct FusedLds<true> {
  union {
    RowsLds r;
    HubLds h;
  };
  __device__ FusedLds() {}
};
template <int G, int V, int OP, bool HAS_VAL, bool ACC = false, bool HUB = false, bool FOLD = false>
__global__ __launch_bounds__(kBlock, fused_waves_per_simd(OP, FOLD)) void spmm_fused(int M, int N, int nbh, int nbu, int rpw, const int *__restrict__ rowptr,
                                                     const int *__restrict__ col, const float *__restrict__ val,
                                                     const float *__restrict__ B, float *__restrict__ C,
                                                     int *__restrict__ E, const UnitTab ut, float *__restrict__ part,
                                                     int *__restrict__ parte, const AccArg aa, const HubArg ha) {
  __shared__ FusedLds<HUB> lds;
  int bx = blockIdx.x;
  if constexpr (HUB) {
    if (bx < nbh) {
      spmm_hub_body<G, V, OP == DGS_MEAN, HAS_VAL, true, kHubBlockFloats>(bx, nbh, lds.h.f, N, col, val, B, C, ha, aa.epi);
      return;
    }
    bx -= nbh;  // nbh is a multiple of 8: block index and XCD keep their relation
  }
  const int ngrid = (int)gridDim.x - (HUB ? nbh : 0);
  if (bx < nbu)
    spmm_units_body<G, V, OP, HAS_VAL, ACC, FOLD>(bx, nbu, lds.r, N, rowptr, col, val, B, C, E, ut, part, parte, aa);
  else {
    // XCD-aware row mapping: workgroups are dealt round-robin to the 8 XCDs (observed: block b -> XCD b % 8), each
    // with a private L2.  Give every XCD a CONTIGUOUS eighth of the row blocks, so that neighbouring rows - which
    // in a locality-preserving ordering share columns - hit the same L2 instead of fetching the same B rows 8x.
    // Pure speed hint: any placement gives the same result.
    int rb = bx - nbu;
#if DGS_XCD_REMAP
    const int nbr = ngrid - nbu;
    const int per = nbr / 8;
    if (rb < per * 8) rb = (rb % 8) * per + rb / 8;
#endif
    spmm_rows_body<G, V, OP, HAS_VAL, false, ACC>(rb, rpw, lds.r, M, N, rowptr, col, val, B, C, E, aa);
  }
}

// ---------------------------------------------------------------------------------------------------------
// Small inputs (the Cora/Citeseer/Pubmed/PPI class: a few 10^4 rows, <= 2.6e5 nnz) finish in a few microseconds,
// so launch count is what matters: ONE launch, row blocks only, every long row reduced by its whole wave in place.
template <int G, int V, int OP, bool HAS_VAL, bool ACC = false>
__global__ __launch_bounds__(kBlock) void spmm_small(int M, int N, int rpw, const int *__restrict__ rowptr,
                                                     const int *__restrict__ col, const float *__restrict__ val,
                                                     const float *__restrict__ B, float *__restrict__ C,
                                                     int *__restrict__ E, const AccArg aa) {
  __shared__ RowsLds lds;
  spmm_rows_body<G, V, OP, HAS_VAL, true, ACC>(blockIdx.x, rpw, lds, M, N, rowptr, col, val, B, C, E, aa);
}

// ---------------------------------------------------------------------------------------------------------
// Strict-order launches (spmm_strict.h): the fused launch with strict unit waves instead of the wave-cooperative tree, and
// the single-launch kernel with its long rows as whole-tile strict units.  No combine.
template <int G, int V, int OP, bool HAS_VAL, int STRICT>
__global__ __launch_bounds__(kBlock, 4) void spmm_fused_strict(int M, int N, int nbu, int rpw, const HubTab ht,
                                                               const int *__restrict__ rowptr, const int *__restrict__ col,
                                                               const float *__restrict__ val, const float *__restrict__ B,
                                                               float *__restrict__ C, const SpmmWs *__restrict__ hdr,
                                                               const int4 *__restrict__ units,
                                                               const StrictPlanHdr *__restrict__ sp) {
  __shared__ union U {
    RowsLds r;
    StrictLds s;
    __device__ U() {}
  } lds;
  if ((int)blockIdx.x < nbu) {
    spmm_units_strict_body<G, V, OP == DGS_MEAN, HAS_VAL, STRICT != 2>(blockIdx.x, nbu, lds.s, N, col, val, B, C, hdr, units, ht, sp);
  } else {
    int rb = blockIdx.x - nbu;
#if DGS_XCD_REMAP
    const int nbr = gridDim.x - nbu;
    const int per = nbr / 8;
    if (rb < per * 8) rb = (rb % 8) * per + rb / 8;
#endif
    spmm_rows_body<G, V, OP, HAS_VAL, false, false, STRICT>(rb, rpw, lds.r, M, N, rowptr, col, val, B, C, nullptr);
  }
}

// The single-launch kernel for inputs that CAN hold a row above the hub threshold (nnz > threshold; sum / mean).  The row waves
// skip such rows and leave their positions in a mask; when all four waves are through, the workgroup chains each of them
// - slice after slice of the feature tile - as the hub workgroup of the general schedule does (strict_hub_coop: three waves
// gather, one chains), in the LDS the row stream no longer needs.  28 KB and the fused HUB kernel's register budget instead
// of 20.5 KB: the inputs below the threshold keep spmm_small as it was.
template <int G, int V, int OP, bool HAS_VAL>
__global__ __launch_bounds__(kBlock) void spmm_small_hub(int M, int N, int rpw, int thub, const int *__restrict__ rowptr,
                                                         const int *__restrict__ col, const float *__restrict__ val,
                                                         const float *__restrict__ B, float *__restrict__ C, const AccArg aa) {
  __shared__ union U {
    RowsLds r;
    HubLds h;
    __device__ U() {}
  } lds;
  __shared__ unsigned hubmask[2 * (kBlock / kWave)];
  if (threadIdx.x < 2 * (kBlock / kWave)) hubmask[threadIdx.x] = 0u;
  __syncthreads();
  spmm_rows_body<G, V, OP, HAS_VAL, true, false, 3>(blockIdx.x, rpw, lds.r, M, N, rowptr, col, val, B, C, nullptr, aa, nullptr, thub,
                                                    hubmask);
  __syncthreads();  // every wave has left the row stream's LDS; the mask is complete
  constexpr int SH = strict_shub(G, V);
#pragma unroll 1
  for (int w = 0; w < 2 * (kBlock / kWave); w++) {
    unsigned m = hubmask[w];  // (block-uniform)
    while (m) {
      const int b = __ffs((int)m) - 1;
      m &= m - 1;
      const int row = (blockIdx.x * (kBlock / kWave) + (w >> 1)) * rpw + (w & 1) * 32 + b;
      const int rs = rowptr[row], len = rowptr[row + 1] - rs;
#pragma unroll 1
      for (int j = 0; j < SH; j++)
        strict_hub_coop<V, G / SH, OP == DGS_MEAN, HAS_VAL, true, kHubBlockFloats>(row, rs, len, blockIdx.y * G * V, j, N, col, val, B,
                                                                               C, lds.h.f, aa.epi);
    }
  }
}

template <int G, int V, int OP, bool HAS_VAL, int STRICT>
__global__ __launch_bounds__(kBlock) void spmm_small_strict(int M, int N, int rpw, const int *__restrict__ rowptr,
                                                            const int *__restrict__ col, const float *__restrict__ val,
                                                            const float *__restrict__ B, float *__restrict__ C) {
  __shared__ RowsLds lds;
  __shared__ StrictLds sl;
  spmm_rows_body<G, V, OP, HAS_VAL, true, false, STRICT>(blockIdx.x, rpw, lds, M, N, rowptr, col, val, B, C, nullptr, AccArg{},
                                                         sl.wave_region(threadIdx.x >> 6));
}

// ---------------------------------------------------------------------------------------------------------
// K3: one wave per entry of the long-row table (launches that do not fold inside the fused kernel).
template <int G, int V, int OP, bool ACC = false>
__global__ __launch_bounds__(kBlock) void spmm_combine(int N, const int *__restrict__ rowptr,
                                                       const int *__restrict__ col, const float *__restrict__ val,
                                                       const float *__restrict__ B, float *__restrict__ C,
                                                       int *__restrict__ E, const UnitTab ut,
                                                       const float *__restrict__ part,
                                                       const int *__restrict__ parte, const AccArg aa, const int skip_hub) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int n_long = *ut.n_long;
  const int wstride = gridDim.x * (kBlock / kWave);
  for (int i = blockIdx.x * (kBlock / kWave) + wave; i < n_long; i += wstride) {
    const int4 d = ut.longrows[i];  // {row, first partial slot, units in the row, 1 = a plan's hub row}
    if (skip_hub && d.w) continue;  // chained whole by the hub blocks of the fused launch: nothing to fold
    fold_row<G, V, OP, ACC, false>(d, lane, N, rowptr, col, val, B, C, E, part, parte, aa);
  }
}

// ---------------------------------------------------------------------------------------------------------
#ifndef DGS_NBU
#define DGS_NBU 1024  // persistent unit blocks of the fused launch
#endif
struct SpmmArgs {
  int64_t M, K, N, nnz;
  const int *rowptr, *col;
  const float *val, *B;
  float *C;
  int *E;
  int tiles;
  void *ws;  // nullptr => single-kernel path
  hipStream_t st;
  int reduce_op;
  // cached plan (dgs_spmm_plan_build): device tables + the counts the host needs to size grids and the workspace
  const struct PlanHdr *plan = nullptr;
  int plan_units = 0, plan_long = 0, plan_pslots = 0, plan_off_long = 0, plan_hub = 0, plan_off_hub = 0;
  int hints = 0;  // DGS_ALG_* bits of the `algorithm` argument
  bool accumulate = false;      // merge into C (and E) instead of overwriting (sum, max, min): see AccArg
  AccArg acc{};
};

// Device-resident header of a cached plan, followed by the tables (all offsets in bytes from the header).
constexpr int kPlanMagic = 0x64677350;  // "dgsP"
struct PlanHdr {
  int magic, version;
  int M, nnz, K;
  int n_units, n_long, n_pslots;
  int ch, t1, tslice, unit;
  int xcd_start[9];     // first unit of each XCD's share of the (sorted) unit table
  int slice_bound[9];   // column-slice boundaries (slice x = columns [b[x], b[x+1]))
  int thub, n_hub;      // rows longer than thub are ALSO listed in the hub table, sorted longest first (sum / mean chain them)
  int xcd_hub[8];       // first hub-row unit of each XCD's share (they sit behind the share's other units)
  int reserved[3];
};
static_assert(sizeof(PlanHdr) <= 256, "plan header must fit its 256-byte slot");

// Column-panel schedule (spmm_panel.h): dense graphs whose dense operand does not fit the L2s.
static inline PanelPlan panel_plan(const SpmmArgs &a, int tiles, int G) {
  PanelPlan P{};
  const Tuning &T = tuning();
  const int force = tune(T.panel, -1);
  // the sweep needs one workgroup per CU, all co-resident: not on a GPU the caller shares with other kernels
  if (force == 0 || !a.ws || (tiles != 1 && G != 64) || G < 8 || a.N % 4 || a.M <= 0 || (a.hints & DGS_ALG_SHARED_GPU)) return P;
  P.nwg = cu_count();
  const bool arg = (a.reduce_op == DGS_MAX || a.reduce_op == DGS_MIN);
  const int64_t W = a.N < 256 ? a.N : 256;  // feature tile per launch (wider operands: one sweep per 256 features)
  const int ebytes = arg ? 6 : 4;  // fp32 value (+ 16-bit arg position | 32-bit arg id)
  int slots = (int)(kPanelAccBytes / (W * ebytes)) & ~1;  // the dispatch rule's calibration (128 KiB of accumulators)
  if (slots > kPanelRMax) slots = kPanelRMax;
  if (slots < 8) return P;
  int rmax = (int)(kPanelLdsBytes / (W * ebytes + kPanelRowState)) & ~1;  // what really fits: accumulators + row state
  if (rmax > kPanelRMax) rmax = kPanelRMax;
  // Worth it when (a) the dense operand overflows the L2s and (b) an XCD's workgroups touch every panel row several
  // times per sweep: reuse = (rows resident per XCD) * (nnz per row) / K = gathered bytes / re-fetched panel bytes, and
  // a row visit still holds a handful of nnz: visit = (nnz per row) * (panel rows) / K.  Measured on MI355X (233 k
  // rows): reuse 6.8 / visit 10 wins 1.13x, 5.6 / 8.4 wins 1.05x, 4.5 / 6.7 loses 1.13x, 4.3 / 13 (min, N = 256) wins
  // 1.22x, 2.8 / 4.2 ties.
  const double bbytes = (double)a.K * W * 4.0;
  const double deg = (double)a.nnz / (double)a.M;
  const double reuse = (P.nwg / 8.0) * slots * deg / (double)(a.K > 0 ? a.K : 1);
  int pkb = tune(T.panel_kb, 6144);
  if (pkb < 1) pkb = 1;
  const int64_t pbytes = (int64_t)pkb * 1024;
  int64_t pc = pbytes / (W * (a.reduce_op == kOpMaskSum ? 8 : 4));  // masked sum gathers grad AND arg-id rows
  if (pc < 64) pc = 64;
  const double visit = deg * (double)pc / (double)(a.K > 0 ? a.K : 1);
  const bool pays = reuse >= 5.5 || (reuse >= 4.0 && visit >= 10.0);
  if (force != 1 && !(bbytes >= 16e6 && pays && a.M >= 4096)) return P;
  P.nsb = (int)((a.M + (int64_t)P.nwg * rmax - 1) / ((int64_t)P.nwg * rmax));
  P.R = (int)((a.M + (int64_t)P.nwg * P.nsb - 1) / ((int64_t)P.nwg * P.nsb));
  P.pcols = (int)pc;
  P.npanels = (int)((a.K + pc - 1) / pc);
  if (P.npanels < 1) P.npanels = 1;
  P.lead = tune(T.panel_lead, 1);
  P.tlong = tune(T.panel_tlong, 4096);
  P.lds = (((size_t)P.R * W * ebytes + 15) & ~size_t(15)) + (size_t)P.R * kPanelRowState;
  P.use = true;
  return P;
}

// Hub threshold of the default sum / mean launches: rows longer than this are chained whole (spmm_hub_body) instead of being
// folded by the fixed tree.  The reference's result is a sequential fp32 chain (include/cuda/spmm_cuda.cuh:27-47), whose own
// rounding error grows like sqrt(len): on the headline graph it stays below 6.3e-6 of the exact sum up to 16384 nnz (5 sigma
// inside the bar), reaches 7.4e-6 at 16 - 32 k (3.8 sigma: not safe over thousands of elements) and 1.2e-5 on the 50 k-nnz rows
// (profiles/r04_chain_error_by_length.txt) - a tree that is closer to the exact sum than that is further than 1e-5 from the
// REFERENCE there.  Above the threshold the chain is reproduced bit for bit; below it the tree is within ~7e-6 of it
// (non-negative data; DGS_ALG_STRICT_SUM chains every row).  Why not lower: a chain runs at ~3 - 5 ns per link, so a row of L
// nnz is an L x 4 ns critical path - 16384 nnz are ~70 us, which a launch over millions of nnz hides, while the 9 - 13 k-nnz
// hub of an arxiv-sized graph (a 48 us call) would not be.
// Two things switch the chains off for a launch: the caller's DGS_ALG_NO_HUB_ROWS hint (it knows the longest row: the launch then
// takes the kernels without the hub role - spmm_small instead of spmm_small_hub, no hub workgroups at the head of the fused grid),
// and the device gate - without an explicit DGS_HUB_CHAIN the chains are on only on a device where dgs_spmm_hub_selftest() has
// compared them with a one-thread-per-element sequential kernel and found them bit-identical (hub_gate(): the hub
// workgroup leans on scheduling behaviour no CPU test can see, so no device runs it unverified by default).
constexpr int kHintForceHub = 0x40000000;  // internal (the self-test itself): default threshold whatever the gate says
constexpr int kHintForceFold = 0x20000000;  // internal (the self-test): fold inside the fused launch whatever the gate says
constexpr int kHintNoFold = 0x10000000;     // internal (the self-test's hub pass): separate combine launch
// What an extern "C" entry lets through from its caller's `algorithm` argument: the documented DGS_ALG_* bits and nothing else -
// the three internal bits above override the device gate, which only the self-test may do.
constexpr int kPublicHints = DGS_ALG_SHARED_GPU | DGS_ALG_STRICT_SUM | DGS_ALG_STRICT_NOFMA | DGS_ALG_NO_HUB_ROWS | DGS_ALG_NO_HUB_COLS;
static inline int public_hints(int algorithm) { return algorithm & kPublicHints; }
int hub_gate();                            // misc.hip: 1 = self-test passed on the current device, 0 = not run, -1 = failed
void hub_gate_set(int state);
int fold_gate();                           // the same for the in-kernel fold of partial rows
void fold_gate_set(int state);
// Fold the partial rows of multi-unit rows INSIDE the fused launch (last-arriving unit wave, spmm_units_body) instead of in a
// combine launch behind it.  OFF unless asked for (round 6, ADVICE r5 / the decision rule of VERDICT r5 #1: the fold stays a default
// only with a hardware measurement fold.on_ms < fold.off_ms, and there is none): DGS_FOLD unset or 0 = the combine launch (the path
// every hardware-verified result of this repo took), DGS_FOLD=1 = fold in the kernel, DGS_FOLD=2 ("auto") = fold in the kernel on a
// device where dgs_spmm_fold_selftest has seen it produce the combine launch's bits - every (G, V) family of partial rows, repeated,
// with the fabric loaded by a streaming kernel.  The hand-over of partial rows between workgroups on different XCDs rests on
// agent-scope stores / loads around an atomic counter (the MI355X guide's R1 form) - memory-system behaviour the plain CPU emulation
// cannot see (tests/emu's relaxed-memory mode models it: sc1 write-through, per-wave store queues, per-XCD dirty lines, per-CU L1).
// The fold's buffer descriptors reach a partial row through a 32-bit byte offset: in-kernel fold only below 2^31 bytes of partial
// rows (20 MB on the headline graph; beyond, the combine launch folds - nothing else changes).
static inline bool fold_fits(int64_t pslots, int64_t N) { return pslots * fold_stride(N) * 4 + 128 < (int64_t(1) << 31); }
static inline bool fold_enabled(int hints) {
  if (hints & kHintNoFold) return false;
  if (hints & kHintForceFold) return true;
  const int e = tuning().fold;
  if (e == kTuneUnset || e == 0) return false;
  return e == 2 ? fold_gate() > 0 : true;
}
static inline int hub_threshold(int hints = 0) {
  if (hints & DGS_ALG_NO_HUB_ROWS) return INT_MAX;
  if (hints & kHintForceHub) return kHubChain;
  const int e = tuning().hub_chain;
  if (e == kTuneUnset) return hub_gate() > 0 ? kHubChain : INT_MAX;
  if (e <= 0 || e > (1 << 24)) return INT_MAX;  // (the class bounds thub << c must stay inside an int)
  return e < kHubChainMin ? kHubChainMin : e;
}
// Threshold a PLAN's hub table is cut with: the compiled-in default (or the explicit DGS_HUB_CHAIN), whatever the device gate says
// at build time - a plan built before the self-test has run (a C caller that never runs it, a build queued during stream capture)
// would otherwise carry n_hub = 0 for good and its planned sums would keep the tree on rows the plan-free calls chain once the gate
// is up.  Whether a LAUNCH uses the table is still decided per call by hub_threshold(a.hints).
static inline int plan_hub_threshold() {
  const int e = tuning().hub_chain;
  if (e == kTuneUnset) return kHubChain;
  if (e <= 0 || e > (1 << 24)) return INT_MAX;
  return e < kHubChainMin ? kHubChainMin : e;
}
// Hub blocks of a launch: a multiple of 8 (XCD mapping), one per task up to four per CU (they come first in the grid: every hub
// chain starts at once and the short ones hand their slots to the unit and row blocks within tens of microseconds)
static inline int hub_blocks(int64_t tasks) {
  int64_t b = (tasks + 7) & ~int64_t(7);
  const int cap = (4 * cu_count() + 7) & ~7;
  return (int)(b < cap ? b : cap);
}

template <int OP>
constexpr bool fold_ok() { return OP != kOpMaskSum; }  // (the in-kernel fold has no masked-sum instantiation)
template <int G, int V, int OP, bool HAS_VAL, bool ACC, bool FOLD>
static void launch_fused_f(const SpmmArgs &a, int nbh, int nbu, int64_t nbr, int rpw, const UnitTab &ut, float *part, int *parte,
                           const HubArg &ha) {
  if constexpr (hub_ok<OP, V, G, ACC>()) {
    if (nbh > 0) {
      hipLaunchKernelGGL((spmm_fused<G, V, OP, HAS_VAL, ACC, true, FOLD>), dim3((unsigned)(nbh + nbu + nbr), (unsigned)a.tiles),
                         dim3(kBlock), 0, a.st, (int)a.M, (int)a.N, nbh, nbu, rpw, a.rowptr, a.col, a.val, a.B, a.C, a.E, ut, part,
                         parte, a.acc, ha);
      return;
    }
  }
  hipLaunchKernelGGL((spmm_fused<G, V, OP, HAS_VAL, ACC, false, FOLD>), dim3((unsigned)(nbu + nbr), (unsigned)a.tiles), dim3(kBlock), 0,
                     a.st, (int)a.M, (int)a.N, 0, nbu, rpw, a.rowptr, a.col, a.val, a.B, a.C, a.E, ut, part, parte, a.acc, HubArg{});
}
// ut.arrive != nullptr (the launcher decided to fold in the kernel: fold_enabled + fold_fits + fold_ok) picks the FOLD = true twin
template <int G, int V, int OP, bool HAS_VAL, bool ACC>
static void launch_fused(const SpmmArgs &a, int nbh, int nbu, int64_t nbr, int rpw, const UnitTab &ut, float *part, int *parte,
                         const HubArg &ha) {
  if constexpr (fold_ok<OP>()) {
    if (ut.arrive != nullptr) {
      launch_fused_f<G, V, OP, HAS_VAL, ACC, true>(a, nbh, nbu, nbr, rpw, ut, part, parte, ha);
      return;
    }
  }
  launch_fused_f<G, V, OP, HAS_VAL, ACC, false>(a, nbh, nbu, nbr, rpw, ut, part, parte, ha);
}

template <int G, int V, int OP, bool HAS_VAL, bool ACC>
static int launch_impl(const SpmmArgs &a) {
  if constexpr (V == 4 && G >= 8 && !ACC) {
    const PanelPlan P = panel_plan(a, a.tiles, G);
    if (P.use) {
      // rows up to tlong nnz: panel sweep; longer rows: the unit path (classify -> unit blocks -> combine)
      const WsLayout L = ws_layout(a.reduce_op, a.N, a.nnz);
      char *w = static_cast<char *>(a.ws);
      SpmmWs *hdr = reinterpret_cast<SpmmWs *>(w);
      int4 *units = reinterpret_cast<int4 *>(w + L.off_units);
      int4 *longrows = reinterpret_cast<int4 *>(w + L.off_long);
      float *part = reinterpret_cast<float *>(w + L.off_part);
      int *parte = reinterpret_cast<int *>(w + L.off_parte);
      UnitTab ut{&hdr->n_units, &hdr->n_long, nullptr, units, longrows};
      if (fill_words(hdr, 0u, sizeof(SpmmWs), a.st) != DGS_OK) return DGS_ELAUNCH;
      const int64_t k0b = (a.M + (int64_t)kBlock * kK0Rows - 1) / ((int64_t)kBlock * kK0Rows);
      int tl = P.tlong > L.ch ? P.tlong : L.ch;  // every long row has >= 2 units => all go through combine
      if (tl > 65534) tl = 65534;  // max keeps 16-bit arg positions (unit lengths never exceed 32768: still >= 2 units)
      int thub = hub_ok<OP, V, G, ACC>() ? hub_threshold(a.hints) : INT_MAX;
      if (thub < tl) thub = tl;  // rows up to tl belong to the panel sweep (one sequential chain per row already)
      const HubTab ht = hub_tab(a.nnz, thub < INT_MAX ? thub : kHubChainMin, a.nnz / kT1 + 2);
      const bool fold = fold_ok<OP>() && fold_enabled(a.hints) && fold_fits(L.max_pslots, a.N);
      if (fold) {
        ut.slot_long = reinterpret_cast<const int *>(w + L.off_slot);
        ut.arrive = reinterpret_cast<int *>(w + L.off_arrive);
        ut.pstride = (int)fold_stride(a.N);
        part = align128(part), parte = align128(parte);
        ut.part_bytes = (unsigned)(L.max_pslots * ut.pstride * 4);
      }
      hipLaunchKernelGGL(spmm_classify, dim3((unsigned)k0b), dim3(kBlock), 0, a.st, (int)a.M, L.ch, tl, thub, ht, a.rowptr, hdr,
                         units, longrows, const_cast<int *>(ut.slot_long), ut.arrive, (int)a.tiles);
      auto kern = spmm_panel<G, OP, HAS_VAL>;
      static std::atomic<bool> attr_set[64];  // per instantiation and device: allow the large dynamic LDS (setting it twice is harmless)
      int dev_id = 0;
      if (hipGetDevice(&dev_id) != hipSuccess || dev_id < 0 || dev_id >= 64) return DGS_ELAUNCH;
      if (!attr_set[dev_id]) {
        if (hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                kPanelLdsBytes) != hipSuccess)
          return DGS_ELAUNCH;
        attr_set[dev_id] = true;
      }
      for (int64_t fb = 0; fb < a.N; fb += 256) {  // one sweep per 256-feature tile, counter re-zeroed in between
        const int W = (int)(a.N - fb < 256 ? a.N - fb : 256);
        if (fb && fill_words(&hdr->arrivals, 0u, sizeof(int), a.st) != DGS_OK) return DGS_ELAUNCH;
        hipLaunchKernelGGL(kern, dim3((unsigned)P.nwg), dim3(kPanelBlock), P.lds, a.st, (int)a.M, W, (int)a.N, P.R, tl,
                           P.pcols, P.npanels, P.nsb, P.lead, a.rowptr, a.col, a.val, a.B + fb, a.C + fb,
                           a.E ? a.E + fb : nullptr, &hdr->arrivals,
                           Epi{a.acc.epi.bias ? a.acc.epi.bias + fb : nullptr, a.acc.epi.rscale, a.acc.epi.relu});
      }
      const int nbu = 1024;
      launch_fused<G, V, OP, HAS_VAL, ACC>(a, thub < INT_MAX ? hub_blocks(2 * cu_count()) : 0, nbu, 0, kRowsPerWave, ut, part, parte,
                                           HubArg{hdr->hub, units, ht, kHubClasses});
      if (!fold) {
        const int64_t cb = (L.max_long + 3) / 4;
        const dim3 g3((unsigned)(cb < 2048 ? (cb < 1 ? 1 : cb) : 2048), (unsigned)a.tiles);
        hipLaunchKernelGGL((spmm_combine<G, V, OP, ACC>), g3, dim3(kBlock), 0, a.st, (int)a.N, a.rowptr, a.col, a.val, a.B,
                           a.C, a.E, ut, part, parte, a.acc, 0);
      }
      return check_launch();
    }
  }
  if (!a.ws) {
    // fewer rows per wave on small inputs: parallelism (>= ~2k waves) matters more than staging efficiency
    constexpr int NGc = kWave / G;
    int rpw = kRowsPerWave;
    while (rpw > NGc && rpw > 4 && (a.M + rpw - 1) / rpw < 2048) rpw >>= 1;
    const int rpb = (kBlock / kWave) * rpw;
    const dim3 grid((unsigned)((a.M + rpb - 1) / rpb), (unsigned)a.tiles);
    if constexpr (hub_ok<OP, V, G, ACC>()) {
      const int thub = hub_threshold(a.hints);
      if (a.nnz > thub) {  // (a row above the threshold needs that many nnz to begin with; callers that know the longest row
                           // say so with DGS_ALG_NO_HUB_ROWS and keep spmm_small)
        hipLaunchKernelGGL((spmm_small_hub<G, V, OP, HAS_VAL>), grid, dim3(kBlock), 0, a.st, (int)a.M, (int)a.N, rpw, thub,
                           a.rowptr, a.col, a.val, a.B, a.C, a.acc);
        return check_launch();
      }
    }
    hipLaunchKernelGGL((spmm_small<G, V, OP, HAS_VAL, ACC>), grid, dim3(kBlock), 0, a.st, (int)a.M, (int)a.N, rpw,
                       a.rowptr, a.col, a.val, a.B, a.C, a.E, a.acc);
    return check_launch();
  }
  // rows per wave: 64 when there are plenty of rows; mid-size graphs (arxiv-shaped: 169 k rows, 6.5 nnz/row) get fewer,
  // so that the chip still sees >= ~8k waves and a group's sequential stream stays a few gather rounds long
  int rpw = kRowsPerWave;
  const int min_waves = tune(tuning().min_waves, 8192);
  while (rpw > 8 && a.M / rpw < min_waves) rpw >>= 1;
  const int rows_per_block = (kBlock / kWave) * rpw;
  const int64_t nbr = (a.M + rows_per_block - 1) / rows_per_block;
  if (a.plan) {
    // cached plan: the unit tables already exist (hub rows cut at column-slice boundaries, sorted by slice and first
    // column, one slice per XCD), so the call is fused + combine; the workspace only holds the partial rows
    const char *pb = reinterpret_cast<const char *>(a.plan);
    const WsLayout L = ws_layout_plan(a.reduce_op, a.N, a.plan_pslots, a.plan_long);
    char *w = static_cast<char *>(a.ws);
    float *part = reinterpret_cast<float *>(w + L.off_part);
    int *parte = reinterpret_cast<int *>(w + L.off_parte);
    const PlanHdr *ph = a.plan;
    const PlanLayout PL = plan_layout(a.nnz);
    UnitTab ut{&ph->n_units, &ph->n_long, ph->xcd_start, reinterpret_cast<const int4 *>(pb + PL.off_units),
               reinterpret_cast<const int4 *>(pb + (a.plan_off_long ? (size_t)a.plan_off_long : PL.off_long))};
    int64_t ub = ((int64_t)a.plan_units + 3) / 4;
    ub = (ub + 7) & ~int64_t(7);  // a multiple of 8 so that the XCD mapping of the unit blocks applies
    int nbu_req = tune(tuning().nbu, DGS_NBU);
    if (nbu_req < 8) nbu_req = 8;  // an override of 0 would leave the units without a single block
    const int nbu_cap = (nbu_req + 7) & ~7;
    const int nbu = (int)(ub < nbu_cap ? (ub < 8 ? 8 : ub) : nbu_cap);
    // hub rows of the plan (longer than the plan's thub): one dense table, longest first, for the sum / mean launches; their
    // units stay in the table (sorted behind the other units of each XCD's share) for every other reduce
    const bool use_hub = hub_ok<OP, V, G, ACC>() && a.plan_hub > 0 && hub_threshold(a.hints) < INT_MAX;
    HubTab ht{};
    const char *hubp = pb + (a.plan_off_hub ? (size_t)a.plan_off_hub : PL.off_hub);
    HubArg ha{&ph->n_hub, reinterpret_cast<const int4 *>(hubp), ht, 1};
    const int nbh = use_hub ? hub_blocks((int64_t)a.plan_hub * strict_shub(G, V)) : 0;
    if (use_hub) ut.xcd_end = ph->xcd_hub;  // the hub rows' units (behind the others of each share) are not walked
    // in-kernel fold: the slot -> long-row map is part of the plan (behind the hub table), the arrival counters are the one piece
    // of the workspace a planned call has to zero (4 bytes per long row: 0.1 MB on the headline graph)
    const bool fold = fold_ok<OP>() && a.plan_long > 0 && fold_enabled(a.hints) && fold_fits(L.max_pslots, a.N);
    if (fold) {
      ut.pstride = (int)fold_stride(a.N);
      part = align128(part), parte = align128(parte);
      ut.part_bytes = (unsigned)(L.max_pslots * ut.pstride * 4);
      ut.slot_long = reinterpret_cast<const int *>(pb + (a.plan_off_hub ? plan_off_slot((size_t)a.plan_off_hub, a.plan_hub) : PL.off_slot));
      ut.arrive = reinterpret_cast<int *>(w + L.off_arrive);
      if (fill_words(ut.arrive, 0u, (size_t)a.plan_long * a.tiles * sizeof(int), a.st) != DGS_OK) return DGS_ELAUNCH;
    }
    launch_fused<G, V, OP, HAS_VAL, ACC>(a, nbh, nbu, nbr, rpw, ut, part, parte, ha);
    if (a.plan_long > 0 && !fold) {
      const int64_t cb = ((int64_t)a.plan_long + 3) / 4;
      const dim3 g3((unsigned)(cb < 2048 ? cb : 2048), (unsigned)a.tiles);
      hipLaunchKernelGGL((spmm_combine<G, V, OP, ACC>), g3, dim3(kBlock), 0, a.st, (int)a.N, a.rowptr, a.col, a.val, a.B,
                         a.C, a.E, ut, part, parte, a.acc, use_hub ? 1 : 0);
    }
    return check_launch();
  }
  const WsLayout L = ws_layout(a.reduce_op, a.N, a.nnz);
  char *w = static_cast<char *>(a.ws);
  SpmmWs *hdr = reinterpret_cast<SpmmWs *>(w);
  int4 *units = reinterpret_cast<int4 *>(w + L.off_units);
  int4 *longrows = reinterpret_cast<int4 *>(w + L.off_long);
  float *part = reinterpret_cast<float *>(w + L.off_part);
  int *parte = reinterpret_cast<int *>(w + L.off_parte);
  UnitTab ut{&hdr->n_units, &hdr->n_long, nullptr, units, longrows};
  if (fill_words(hdr, 0u, sizeof(SpmmWs), a.st) != DGS_OK) return DGS_ELAUNCH;
  const int64_t k0b = (a.M + (int64_t)kBlock * kK0Rows - 1) / ((int64_t)kBlock * kK0Rows);
  const int thub = hub_ok<OP, V, G, ACC>() ? hub_threshold(a.hints) : INT_MAX;
  const HubTab ht = hub_tab(a.nnz, thub < INT_MAX ? thub : kHubChainMin, a.nnz / kT1 + 2);
  const bool fold = fold_ok<OP>() && fold_enabled(a.hints) && fold_fits(L.max_pslots, a.N);  // (the classify pass fills the slot map and zeroes the counters of the rows it lists)
  if (fold) {
    ut.slot_long = reinterpret_cast<const int *>(w + L.off_slot);
    ut.arrive = reinterpret_cast<int *>(w + L.off_arrive);
    ut.pstride = (int)fold_stride(a.N);
    part = align128(part), parte = align128(parte);
    ut.part_bytes = (unsigned)(L.max_pslots * ut.pstride * 4);
  }
  hipLaunchKernelGGL(spmm_classify, dim3((unsigned)k0b), dim3(kBlock), 0, a.st, (int)a.M, L.ch, kT2, thub, ht, a.rowptr, hdr,
                     units, longrows, const_cast<int *>(ut.slot_long), ut.arrive, (int)a.tiles);
  // unit / multi counts live on the device: a bounded number of persistent unit blocks stride over the table
  const int64_t ub = (L.max_units + 3) / 4;
  int nbu_cap = tune(tuning().nbu, DGS_NBU);
  if (nbu_cap < 1) nbu_cap = 1;
  const int nbu = (int)(ub < nbu_cap ? (ub < 1 ? 1 : ub) : nbu_cap);
  // (the hub count lives on the device: two hub workgroups per CU are launched whenever hub chains are on; without hub rows
  // they read six zeros and leave)
  launch_fused<G, V, OP, HAS_VAL, ACC>(a, thub < INT_MAX ? hub_blocks(2 * cu_count()) : 0, nbu, nbr, rpw, ut, part, parte,
                                       HubArg{hdr->hub, units, ht, kHubClasses});
  // combine: one wave per multi-unit row (unless the unit waves fold the rows themselves)
  if (!fold) {
    const int64_t cb = (L.max_long + 3) / 4;
    const dim3 g3((unsigned)(cb < 2048 ? (cb < 1 ? 1 : cb) : 2048), (unsigned)a.tiles);
    hipLaunchKernelGGL((spmm_combine<G, V, OP, ACC>), g3, dim3(kBlock), 0, a.st, (int)a.N, a.rowptr, a.col, a.val, a.B, a.C,
                       a.E, ut, part, parte, a.acc, 0);
  }
  return check_launch();
}

// The strict schedule runs over a cached plan's strict table (built with the default class thresholds) unless an experiment
// override moved those thresholds.
static inline bool strict_over_plan_ok() { return tuning().strict_mid == kTuneUnset && tuning().strict_hub == kTuneUnset; }

#if defined(DGS_TU_STRICT)
// Strict-order sum / mean (spmm_strict.h).  fill + classify_strict + ONE fused launch (no combine); dense graphs keep the
// column-panel sweep for rows up to tlong nnz (its per-row accumulator is a sequential fmaf chain already) and send only
// the longer rows through strict unit waves.
template <int G, int V, int OP, bool HAS_VAL, int STRICT>
static int launch_strict(const SpmmArgs &a) {
  static_assert(OP == DGS_SUM || OP == DGS_MEAN, "strict order exists for sum and mean");
  if (!a.ws) {
    constexpr int NGc = kWave / G;
    int rpw = kRowsPerWave;
    while (rpw > NGc && rpw > 4 && (a.M + rpw - 1) / rpw < 2048) rpw >>= 1;
    const int rpb = (kBlock / kWave) * rpw;
    const dim3 grid((unsigned)((a.M + rpb - 1) / rpb), (unsigned)a.tiles);
    hipLaunchKernelGGL((spmm_small_strict<G, V, OP, HAS_VAL, STRICT>), grid, dim3(kBlock), 0, a.st, (int)a.M, (int)a.N, rpw,
                       a.rowptr, a.col, a.val, a.B, a.C);
    return check_launch();
  }
  if (a.plan) {
    // over a cached plan (round 5): the plan carries every row > T1 sorted longest first with the sizes of the
    // three length classes (spmm_plan.hip: plan_strict_*), so the call is ONE launch - no memset, no classify pass, no workspace
    int nbu_req = tune(tuning().strict_nbu, 8 * cu_count());
    if (nbu_req < 8) nbu_req = 8;
    const int nbu = (nbu_req + 7) & ~7;
    int rpw = kRowsPerWave;
    const int min_waves = tune(tuning().min_waves, 8192);
    while (rpw > 8 && a.M / rpw < min_waves) rpw >>= 1;
    const int rows_per_block = (kBlock / kWave) * rpw;
    const int64_t nbr = (a.M + rows_per_block - 1) / rows_per_block;
    const char *pb = reinterpret_cast<const char *>(a.plan);
    const PlanLayout PL = plan_layout(a.nnz);
    const size_t off_strict = a.plan_off_hub ? plan_off_strict(plan_off_slot((size_t)a.plan_off_hub, a.plan_hub), a.plan_pslots)
                                             : PL.off_strict;
    const StrictPlanHdr *sp = reinterpret_cast<const StrictPlanHdr *>(pb + off_strict);
    hipLaunchKernelGGL((spmm_fused_strict<G, V, OP, HAS_VAL, STRICT>), dim3((unsigned)(nbr + nbu), (unsigned)a.tiles),
                       dim3(kBlock), 0, a.st, (int)a.M, (int)a.N, nbu, rpw, HubTab{}, a.rowptr, a.col, a.val, a.B, a.C,
                       (const SpmmWs *)nullptr, reinterpret_cast<const int4 *>(sp + 1), sp);
    return check_launch();
  }
  const WsLayout L = ws_layout(a.reduce_op, a.N, a.nnz);
  char *w = static_cast<char *>(a.ws);
  SpmmWs *hdr = reinterpret_cast<SpmmWs *>(w);
  int4 *units = reinterpret_cast<int4 *>(w + L.off_units);
  // (DGS_STRICT_MID / _HUB: experiment overrides of the slicing thresholds; the table capacities assume hub >= kStrictHub)
  int tmid = tune(tuning().strict_mid, kStrictMid), thub = tune(tuning().strict_hub, kStrictHub);
  if (thub < (strict_coop(G, V) ? kStrictMid : kStrictHub)) thub = strict_coop(G, V) ? kStrictMid : kStrictHub;
  if (tmid < kStrictMid) tmid = kStrictMid;
  if (tmid > thub) tmid = thub;
  if (fill_words(hdr, 0u, sizeof(SpmmWs), a.st) != DGS_OK) return DGS_ELAUNCH;
  const int64_t k0b = (a.M + (int64_t)kBlock * kK0Rows - 1) / ((int64_t)kBlock * kK0Rows);
  // unit blocks: first in the grid (the long chains must start first), twice as many as fit the chip at once (4 workgroups
  // per CU): the later ones take over as the early ones run out of units, and the row blocks follow as those drain.
  // Measured on the headline graph: 512 blocks 0.84 ms, 1024 0.67, 2048 0.58, 4096 0.58, 16384 0.61
  int nbu_req = tune(tuning().strict_nbu, 8 * cu_count());
  if (nbu_req < 8) nbu_req = 8;
  const int nbu = (nbu_req + 7) & ~7;  // a multiple of 8: one share per XCD
  if constexpr (V == 4 && G >= 8 && STRICT == 1) {
    const PanelPlan P = panel_plan(a, a.tiles, G);
    if (P.use) {
      int tl = P.tlong > kStrictHub ? P.tlong : kStrictHub;
      if (tl > 65534) tl = 65534;
      const HubTab ht = hub_tab(a.nnz, tl, a.nnz / kT1 + 2);
      hipLaunchKernelGGL(spmm_classify_strict, dim3((unsigned)k0b), dim3(kBlock), 0, a.st, (int)a.M, tl, tl, tl, ht, a.rowptr,
                         hdr, units);
      auto kern = spmm_panel<G, OP, HAS_VAL>;
      static std::atomic<bool> attr_set[64];
      int dev_id = 0;
      if (hipGetDevice(&dev_id) != hipSuccess || dev_id < 0 || dev_id >= 64) return DGS_ELAUNCH;
      if (!attr_set[dev_id]) {
        if (hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                kPanelLdsBytes) != hipSuccess)
          return DGS_ELAUNCH;
        attr_set[dev_id] = true;
      }
      for (int64_t fb = 0; fb < a.N; fb += 256) {
        const int W = (int)(a.N - fb < 256 ? a.N - fb : 256);
        if (fb && fill_words(&hdr->arrivals, 0u, sizeof(int), a.st) != DGS_OK) return DGS_ELAUNCH;
        hipLaunchKernelGGL(kern, dim3((unsigned)P.nwg), dim3(kPanelBlock), P.lds, a.st, (int)a.M, W, (int)a.N, P.R, tl,
                           P.pcols, P.npanels, P.nsb, P.lead, a.rowptr, a.col, a.val, a.B + fb, a.C + fb,
                           (int *)nullptr, &hdr->arrivals, Epi{});
      }
      hipLaunchKernelGGL((spmm_fused_strict<G, V, OP, HAS_VAL, STRICT>), dim3((unsigned)nbu, (unsigned)a.tiles), dim3(kBlock),
                         0, a.st, (int)a.M, (int)a.N, nbu, kRowsPerWave, ht, a.rowptr, a.col, a.val, a.B, a.C, hdr, units,
                         (const StrictPlanHdr *)nullptr);
      return check_launch();
    }
  }
  int rpw = kRowsPerWave;
  const int min_waves = tune(tuning().min_waves, 8192);
  while (rpw > 8 && a.M / rpw < min_waves) rpw >>= 1;
  const int rows_per_block = (kBlock / kWave) * rpw;
  const int64_t nbr = (a.M + rows_per_block - 1) / rows_per_block;
  const HubTab ht = hub_tab(a.nnz, thub, a.nnz / kT1 + 2);
  hipLaunchKernelGGL(spmm_classify_strict, dim3((unsigned)k0b), dim3(kBlock), 0, a.st, (int)a.M, kT1, tmid, thub, ht, a.rowptr,
                     hdr, units);
  hipLaunchKernelGGL((spmm_fused_strict<G, V, OP, HAS_VAL, STRICT>), dim3((unsigned)(nbr + nbu), (unsigned)a.tiles),
                     dim3(kBlock), 0, a.st, (int)a.M, (int)a.N, nbu, rpw, ht, a.rowptr, a.col, a.val, a.B, a.C, hdr, units,
                     (const StrictPlanHdr *)nullptr);
  return check_launch();
}

template <int G, int V, int OP>
static int dispatch_strict_val(const SpmmArgs &a) {
  const bool nofma = (a.hints & DGS_ALG_STRICT_NOFMA) != 0;
  if (a.val) return nofma ? launch_strict<G, V, OP, true, 2>(a) : launch_strict<G, V, OP, true, 1>(a);
  return launch_strict<G, V, OP, false, 1>(a);  // weight 1: fmaf(1, x, acc) == acc + x, one variant serves both
}
template <int V>
static int dispatch_strict(int G, const SpmmArgs &a) {
  const bool mean = a.reduce_op == DGS_MEAN;
  switch (G) {
#define DGS_STRICT_CASE(g) case g: return mean ? dispatch_strict_val<g, V, DGS_MEAN>(a) : dispatch_strict_val<g, V, DGS_SUM>(a);
    DGS_STRICT_CASE(1) DGS_STRICT_CASE(2) DGS_STRICT_CASE(4) DGS_STRICT_CASE(8) DGS_STRICT_CASE(16) DGS_STRICT_CASE(32)
    DGS_STRICT_CASE(64)
#undef DGS_STRICT_CASE
  }
  return DGS_EINVAL;
}
#endif  // DGS_TU_STRICT

template <int G, int V, int OP, bool HAS_VAL>
static int launch_all(const SpmmArgs &a) {
  if (a.accumulate) {  // merge into C / (C, E) (sum, max, min; never the column-panel sweep)
    if constexpr (OP == DGS_SUM || OP == DGS_MAX || OP == DGS_MIN) return launch_impl<G, V, OP, HAS_VAL, true>(a);
    else return DGS_EINVAL;
  }
  return launch_impl<G, V, OP, HAS_VAL, false>(a);
}

template <int G, int V, int OP>
static int dispatch_val(const SpmmArgs &a) {
  return a.val ? launch_all<G, V, OP, true>(a) : launch_all<G, V, OP, false>(a);
}

// The kernels are instantiated in three translation units so that the build parallelises
// (spmm_v4a.hip: V=4 sum/mean/masked-sum, spmm_v4b.hip: V=4 max/min, spmm_v1.hip: V=1 everything).
template <int G, int V>
static int dispatch_op(const SpmmArgs &a) {
  switch (a.reduce_op) {
#if !defined(DGS_TU_ARG_ONLY)
    case DGS_SUM: return dispatch_val<G, V, DGS_SUM>(a);
    case DGS_MEAN: return dispatch_val<G, V, DGS_MEAN>(a);
    case kOpMaskSum: return dispatch_val<G, V, kOpMaskSum>(a);
#endif
#if !defined(DGS_TU_SUM_ONLY)
    case DGS_MAX: return dispatch_val<G, V, DGS_MAX>(a);
    case DGS_MIN: return dispatch_val<G, V, DGS_MIN>(a);
#endif
  }
  return DGS_EINVAL;
}

template <int V>
static int dispatch_g(int G, const SpmmArgs &a) {
  switch (G) {
    case 1: return dispatch_op<1, V>(a);
    case 2: return dispatch_op<2, V>(a);
    case 4: return dispatch_op<4, V>(a);
    case 8: return dispatch_op<8, V>(a);
    case 16: return dispatch_op<16, V>(a);
    case 32: return dispatch_op<32, V>(a);
    case 64: return dispatch_op<64, V>(a);
  }
  return DGS_EINVAL;
}

// Inputs this small finish in a few microseconds: launch count dominates, so they take the single-launch path.
static inline bool tiny_problem(int64_t M, int64_t nnz) { return nnz <= (1 << 18) && M <= (1 << 16); }

// one entry per translation unit
int spmm_run_v4_sum(int G, const SpmmArgs &a);  // V=4: sum, mean, masked sum
int spmm_run_v4_arg(int G, const SpmmArgs &a);  // V=4: max, min
int spmm_run_v1(int G, const SpmmArgs &a);      // V=1: all ops
int spmm_run_strict(int G, int V, const SpmmArgs &a);  // strict-order sum / mean (spmm_strict.hip)

}  // namespace dgs
