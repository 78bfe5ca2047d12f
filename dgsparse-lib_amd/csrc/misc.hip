// misc.hip -- row gather / scatter-add (halo pack / unpack for the multi-GPU path), version/info entry
// points, and the GE-SpMM / SDDMM compatibility shims (reference src/ge-spmm/gespmm.h:32-41,
// src/sddmm/sddmm.h:10) over the dgs_* entry points.
#include <stdlib.h>

#include <atomic>
#include <mutex>

#include "dgs_common.h"

namespace dgs {

// ---- clearing (dgs_common.h) --------------------------------------------------------------------------------------------------
static __global__ __launch_bounds__(kBlock) void fill_words_kernel(uint32_t *__restrict__ p, uint32_t word, int64_t words, int64_t pieces) {
  const int64_t n = (int64_t)gridDim.x * kBlock, t = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  const int4 w = make_int4((int)word, (int)word, (int)word, (int)word);
  for (int64_t i = t; i < pieces; i += n) reinterpret_cast<int4 *>(p)[i] = w;
  for (int64_t i = 4 * pieces + t; i < words; i += n) p[i] = word;
}
int fill_words(void *p, uint32_t word, size_t bytes, hipStream_t st) {
  if (bytes == 0) return DGS_OK;
#ifdef DGS_HOST_EMU  // (the emulation has no graphs, and its memset is the host's: words of four equal bytes)
  return hipMemsetAsync(p, (int)(word & 0xff), bytes, st) == hipSuccess ? DGS_OK : DGS_ELAUNCH;
#endif
  const int64_t words = (int64_t)(bytes / 4), pieces = is_aligned16(p) ? words / 4 : 0, work = pieces ? pieces : words;
  const int64_t blocks = (work + kBlock - 1) / kBlock;
  hipLaunchKernelGGL(fill_words_kernel, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(kBlock), 0, st, static_cast<uint32_t *>(p), word, words, pieces);
  return check_launch();
}

// ---- process-wide tuning snapshot + per-device facts (the only global state of the library; see dgs_common.h) -------------
// Every publish is a fresh heap snapshot that is never written again and never freed (64 bytes per dgs_reload_tuning(), a
// tests-only call): a launch that holds `const Tuning &` keeps valid, unchanging values however many reloads follow (
// two alternating static buffers were overwritten in place by the second reload).
static std::atomic<const Tuning *> g_tuning_cur{nullptr};
static std::mutex g_tuning_mu;
static std::once_flag g_tuning_once;
static void tuning_read(Tuning &t) {
  auto rd = [](const char *k) {
    const char *v = getenv(k);
    return (v && *v) ? atoi(v) : kTuneUnset;
  };
  t.panel = rd("DGS_PANEL");
  t.panel_kb = rd("DGS_PANEL_KB");
  t.panel_lead = rd("DGS_PANEL_LEAD");
  t.panel_tlong = rd("DGS_PANEL_TLONG");
  t.min_waves = rd("DGS_MIN_WAVES");
  t.nbu = rd("DGS_NBU");
  t.strict_mid = rd("DGS_STRICT_MID");
  t.strict_hub = rd("DGS_STRICT_HUB");
  t.strict_nbu = rd("DGS_STRICT_NBU");
  t.sddmm_fused = rd("DGS_SDDMM_FUSED");
  t.plan_tslice = rd("DGS_PLAN_TSLICE");
  t.plan_unit = rd("DGS_PLAN_UNIT");
  t.plan_ch = rd("DGS_PLAN_CH");
  t.plan_nocut = rd("DGS_PLAN_NOCUT");
  t.hub_chain = rd("DGS_HUB_CHAIN");
  t.fold = rd("DGS_FOLD");
}
static void tuning_publish() {
  std::lock_guard<std::mutex> lk(g_tuning_mu);
  Tuning *next = new Tuning;
  tuning_read(*next);
  g_tuning_cur.store(next, std::memory_order_release);
}
const Tuning &tuning() {
  std::call_once(g_tuning_once, tuning_publish);
  return *g_tuning_cur.load(std::memory_order_acquire);
}
int cu_count() {
  static std::atomic<int> n[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int v = n[dev].load(std::memory_order_relaxed);
  if (!v) {
    hipDeviceProp_t prop;
    v = (hipGetDeviceProperties(&prop, dev) == hipSuccess && prop.multiProcessorCount > 0) ? prop.multiProcessorCount : 256;
    n[dev].store(v, std::memory_order_relaxed);
  }
  return v;
}

// Device gate of the default hub chains (spmm_impl.h hub_threshold): what dgs_spmm_hub_selftest found on each device.
static std::atomic<int> g_hub_gate[64];
int hub_gate() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 0;
  return g_hub_gate[dev].load(std::memory_order_acquire);
}
void hub_gate_set(int state) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return;
  g_hub_gate[dev].store(state, std::memory_order_release);
}
static std::atomic<int> g_fold_gate[64];
int fold_gate() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 0;
  return g_fold_gate[dev].load(std::memory_order_acquire);
}
void fold_gate_set(int state) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return;
  g_fold_gate[dev].store(state, std::memory_order_release);
}

// One row per G-lane group, V floats per lane: dst[i,:] = src[ids[i],:]
template <int V>
__global__ __launch_bounds__(kBlock) void gather_rows_kernel(int64_t n_ids, int N, const int *__restrict__ ids,
                                                             const float *__restrict__ src,
                                                             float *__restrict__ dst) {
  const int lanes = (N + V - 1) / V;  // lanes needed per row
  const int64_t t = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  const int64_t i = t / lanes;
  const int f = (int)(t % lanes) * V;
  if (i >= n_ids) return;
  float x[V];
  load_vec<V>(src + (int64_t)ids[i] * N + f, x);
  store_vec<V>(dst + i * N + f, x);
}

// N == 1 (a permutation of a value array, e.g. CSR -> CSC order of the edge values): 4 elements per thread, so that
// four independent random reads are in flight per lane and the ids / results move as 16-byte vectors.
__global__ __launch_bounds__(kBlock) void gather_scalar_kernel(int64_t n, const int *__restrict__ ids,
                                                               const float *__restrict__ src,
                                                               float *__restrict__ dst) {
  const int64_t i = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * 4;
  if (i + 3 < n) {
    const dgs_i4 id = __builtin_nontemporal_load(reinterpret_cast<const dgs_i4 *>(ids + i));
    const float a = src[id[0]], b = src[id[1]], c = src[id[2]], d = src[id[3]];
    float o[4] = {a, b, c, d};
    store_vec_stream<4>(dst + i, o);
  } else {
    for (int64_t k = i; k < n; k++) dst[k] = src[ids[k]];
  }
}

template <int V>
__global__ __launch_bounds__(kBlock) void scatter_add_rows_kernel(int64_t n_ids, int N, const int *__restrict__ ids,
                                                                  const float *__restrict__ src,
                                                                  float *__restrict__ dst) {
  const int lanes = (N + V - 1) / V;
  const int64_t t = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  const int64_t i = t / lanes;
  const int f = (int)(t % lanes) * V;
  if (i >= n_ids) return;
  float x[V], y[V];
  float *d = dst + (int64_t)ids[i] * N + f;
  load_vec<V>(src + i * N + f, x);
  load_vec<V>(d, y);
#pragma unroll
  for (int v = 0; v < V; v++) y[v] += x[v];
  store_vec<V>(d, y);
}

// ids[i] = map[ids[i]] for ids[i] >= 0 (negative ids - "no arg" - stay): 4 ids per thread
__global__ __launch_bounds__(kBlock) void relabel_kernel(int64_t n, int *__restrict__ ids, const int *__restrict__ map) {
  const int64_t i = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * 4;
  if (i + 3 < n && (reinterpret_cast<uintptr_t>(ids) & 15u) == 0) {
    dgs_i4 v = *reinterpret_cast<const dgs_i4 *>(ids + i);
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = v[k] >= 0 ? map[v[k]] : v[k];
    *reinterpret_cast<dgs_i4 *>(ids + i) = v;
  } else {
    for (int64_t k = i; k < n && k < i + 4; k++) ids[k] = ids[k] >= 0 ? map[ids[k]] : ids[k];
  }
}

}  // namespace dgs

using namespace dgs;

extern "C" int dgs_relabel_i32(int64_t n, int32_t *ids, const int32_t *map, dgsStream_t stream) {
  if (n < 0) return DGS_EINVAL;
  if (n == 0) return DGS_OK;
  if (!ids || !map) return DGS_EINVAL;
  const int64_t blocks = (n + 4 * kBlock - 1) / (4 * kBlock);
  hipLaunchKernelGGL(relabel_kernel, dim3((unsigned)blocks), dim3(kBlock), 0, static_cast<hipStream_t>(stream), n, ids, map);
  return check_launch();
}

extern "C" int dgs_version(void) { return 1005; }  // 1.1: cached plans, accumulating SpMM, scheduling hints, relabel; 1.2: strict-order bits, dgs_spmm_csr_ex_f32 (epilogue), dgs_sddmm_csr_plan_f32, non-blocking plan helpers; 1.3: accumulating min, min merge / redo, non-finite detector; 1.4 (rounds 4 / 5): hub threshold / tuning reload, the device gate (dgs_spmm_hub_selftest*, _hub_gate, _fold_gate), DGS_ALG_NO_HUB_ROWS / _COLS, strict bits over a plan, dgs_spmm_csr_acc_min_around_f32; 1.5 (round 6): dgs_spmm_fold_selftest / _selftest_detail / _selftest_families, the in-kernel fold opt-in (DGS_FOLD=1 | 2)
extern "C" const char *dgs_arch(void) { return "gfx950"; }
extern "C" const char *dgs_strerror(int code) {
  switch (code) {
    case DGS_OK: return "ok";
    case DGS_EINVAL: return "invalid argument";
    case DGS_EWORKSPACE: return "workspace too small";
    case DGS_ELAUNCH: return "kernel launch failed";
    case DGS_ERANGE: return "size exceeds int32 CSR indexing";
  }
  return "unknown error";
}

extern "C" int dgs_gather_rows_f32(int64_t n_ids, int64_t N, const int32_t *ids, const float *src, float *dst,
                                   dgsStream_t stream) {
  if (n_ids < 0 || N < 0 || N >= INT32_MAX) return DGS_EINVAL;
  if (n_ids == 0 || N == 0) return DGS_OK;
  if (!ids || !src || !dst) return DGS_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (N == 1 && is_aligned16(ids) && is_aligned16(dst)) {
    const int64_t threads = (n_ids + 3) / 4;
    hipLaunchKernelGGL(gather_scalar_kernel, dim3((unsigned)((threads + kBlock - 1) / kBlock)), dim3(kBlock), 0, st, n_ids,
                       ids, src, dst);
    return check_launch();
  }
  const bool v4 = (N % 4 == 0) && is_aligned16(src) && is_aligned16(dst);
  const int64_t lanes = v4 ? N / 4 : N;
  const dim3 grid((unsigned)((n_ids * lanes + kBlock - 1) / kBlock));
  if (v4)
    hipLaunchKernelGGL((gather_rows_kernel<4>), grid, dim3(kBlock), 0, st, n_ids, (int)N, ids, src, dst);
  else
    hipLaunchKernelGGL((gather_rows_kernel<1>), grid, dim3(kBlock), 0, st, n_ids, (int)N, ids, src, dst);
  return check_launch();
}

extern "C" int dgs_scatter_add_rows_f32(int64_t n_ids, int64_t N, const int32_t *ids, const float *src, float *dst,
                                        dgsStream_t stream) {
  if (n_ids < 0 || N < 0 || N >= INT32_MAX) return DGS_EINVAL;
  if (n_ids == 0 || N == 0) return DGS_OK;
  if (!ids || !src || !dst) return DGS_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool v4 = (N % 4 == 0) && is_aligned16(src) && is_aligned16(dst);
  const int64_t lanes = v4 ? N / 4 : N;
  const dim3 grid((unsigned)((n_ids * lanes + kBlock - 1) / kBlock));
  if (v4)
    hipLaunchKernelGGL((scatter_add_rows_kernel<4>), grid, dim3(kBlock), 0, st, n_ids, (int)N, ids, src, dst);
  else
    hipLaunchKernelGGL((scatter_add_rows_kernel<1>), grid, dim3(kBlock), 0, st, n_ids, (int)N, ids, src, dst);
  return check_launch();
}

// ---- compatibility shims: same signatures as the reference's standalone C libraries, default stream ----
extern "C" void gespmmCsrSpMM(const struct SpMatCsrDescr_t A, float *B, const int N, float *C, bool transpose_BC,
                              enum gespmmAlg_t alg) {
  (void)alg;  // all algorithm ids share the algorithm-0 numerics here
  if (!transpose_BC) return;  // column-major B/C is out of scope
  int64_t nnz = A.nnz;
  if (nnz < 0) {  // gespmm.h semantics: nnz < 0 means "read indptr[nrow]"
    int last = 0;
    if (hipMemcpy(&last, A.indptr + A.nrow, sizeof(int), hipMemcpyDeviceToHost) != hipSuccess) return;
    nnz = last;
  }
  // The reference entry point owns no workspace argument: take it from the stream-ordered allocator on the
  // default stream (no host synchronisation; cf. the per-call cudaMalloc in the reference's csr2cscKernel).
  const size_t wsb = dgs_spmm_csr_workspace_bytes(DGS_SUM, A.nrow, N, nnz);
  void *ws = nullptr;
  if (wsb && hipMallocAsync(&ws, wsb, nullptr) != hipSuccess) return;
  dgs_spmm_csr_f32(DGS_SUM, A.nrow, A.ncol, N, nnz, A.indptr, A.indices, A.data, B, C, nullptr, 0, ws, wsb, nullptr);
  if (ws) (void)hipFreeAsync(ws, nullptr);
}
extern "C" void spmm_cuda(int nrowA, int ncolB, int *rowptr, int *colind, float *values, float *dense, float *out) {
  struct SpMatCsrDescr_t A = {nrowA, 0, -1, rowptr, colind, values};
  A.ncol = INT32_MAX - 1;
  gespmmCsrSpMM(A, dense, ncolB, out, true, GESPMM_ALG_DEFAULT);
}
extern "C" void spmm_cuda_no_edge_value(int nrowA, int ncolB, int *rowptr, int *colind, float *values, float *dense,
                                        float *out) {
  (void)values;
  struct SpMatCsrDescr_t A = {nrowA, INT32_MAX - 1, -1, rowptr, colind, nullptr};
  gespmmCsrSpMM(A, dense, ncolB, out, true, GESPMM_ALG_DEFAULT);
}
extern "C" void sddmm_cuda_csr(int m, int k, int nnz, int *rowptr, int *colind, float *D1, float *D2, float *out) {
  dgs_sddmm_csr_f32(DGS_SUM, m, INT32_MAX - 1, k, nnz, rowptr, colind, D1, D2, out, nullptr);
}
extern "C" void sddmm_cuda_coo(int k, int nnz, int *rowind, int *colind, float *D1, float *D2, float *out) {
  dgs_sddmm_coo_f32(k, nnz, rowind, colind, D1, D2, out, nullptr);
}
// src/ge-spmm/gespmm.cc:13-24: the reference's kernel selector.  Every id runs the same schedule here.
extern "C" enum gespmmAlg_t gespmmAlgSel(int dense_ncol, bool transpose_BC) {
  if (!transpose_BC) return GESPMM_ALG_PARREDUCE_ROWBALANCE_NON_TRANSPOSE;
  if (dense_ncol >= 32) return GESPMM_ALG_ROWCACHING_ROWBALANCE;
  return dense_ncol > 4 ? GESPMM_ALG_SEQREDUCE_ROWBALANCE : GESPMM_ALG_PARREDUCE_ROWBALANCE;
}
// src/ge-spmm/gespmm.h:64-84: the per-algorithm entry points (row-major B/C).  The nnz-balanced variants of the
// reference ACCUMULATE into a caller-zeroed C with atomics (example/ge-spmm/spmm.cu:182); these overwrite C, which
// is the same result under that calling convention.
#define DGS_GESPMM_ALIAS(name)                                                                       \
  extern "C" void name(const struct SpMatCsrDescr_t A, const float *B, const int N, float *C) {     \
    gespmmCsrSpMM(A, const_cast<float *>(B), N, C, true, GESPMM_ALG_DEFAULT);                        \
  }
DGS_GESPMM_ALIAS(csrspmm_parreduce_rowbalance)
DGS_GESPMM_ALIAS(csrspmm_parreduce_nnzbalance)
DGS_GESPMM_ALIAS(csrspmm_seqreduce_rowbalance)
DGS_GESPMM_ALIAS(csrspmm_seqreduce_nnzbalance)
DGS_GESPMM_ALIAS(csrspmm_rowcaching_rowbalance)
DGS_GESPMM_ALIAS(csrspmm_rowcaching_nnzbalance)

extern "C" void dgs_reload_tuning(void) {
  dgs::tuning();  // make sure the first snapshot exists, then publish a fresh one beside it (readers keep a valid pointer)
  dgs::tuning_publish();
}
