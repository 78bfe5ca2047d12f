// rms_norm.hip -- root-mean-square norm with the residual's addition in front of it, its backward pass, and a form whose output leaves in
// 8-bit floating point with a scale for each row and block of 128 columns.
//
//   s = x + residual, rounded once to the type of x: it is what the next layer reads as its residual, and what the norm is taken of (so
//       that forward and backward see the same values)
//   y = s r w,  r = 1 / sqrt(mean(s^2) + eps)
//   dx = dresidual = r (w dy) - s r^3 mean(s w dy) + ds ;  dw = sum over rows of dy s r
//       taken as r (w dy - (s r) (r mean(s w dy))) + ds: every factor is an ordinary number where s and its squares' sum are, while r^3 by itself
//       leaves the range of 32 bits for rows beyond 1e13 or (with an eps next to nothing) below 1e-13
//
// Bound: HBM.  Forward reads 2 rows and writes 2, backward reads 3 and writes 1; a row is read once and stays in registers between its
// reduction and its use (NV 16-byte vectors per lane).  Row statistics and dw are sums in 32 bits.
// Measured (kernel time; a large copy runs at 5.1 TB/s):  8192 x 4096 bf16 forward 50 us (5.3 TB/s), backward 55 (4.9) and 10 for dw's join;
// 169343 x 128 fp32 57 (6.1, part of it out of the last cache), 73 (4.7) and 11;  8-bit output, 8191 x 5120 fp16, 59 us (5.0 TB/s).
#include "dense_common.h"

namespace dgs {

// A row is worked by G lanes, each holding NV vectors: vector j of lane l starts at element (l + j G) kVec.  NV = 0: rows longer than the
// registers take; s is read again in the second pass.
template <typename T, bool VECTOR, int G, int NV, bool RES, bool FP8>
__global__ __launch_bounds__(kBlock) void rms_norm_kernel(int64_t rows, int D, const T *__restrict__ x, int64_t ldx,
                                                          const T *__restrict__ residual, int64_t ldr, const T *__restrict__ w, float eps,
                                                          T *__restrict__ y, T *__restrict__ s_out, uint8_t *__restrict__ q,
                                                          float *__restrict__ scales) {
  constexpr int V = kVec<T>;
  constexpr int kKeep = NV ? NV : 1, kUnroll = kKeep;
  __shared__ float red[4];
  const int lane = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * (kBlock / G) + threadIdx.x / G;
  if (G <= 64 && row >= rows) return;  // (G = 256: one row a workgroup, the grid has exactly `rows` of them)
  const T *xr = x + row * ldx, *rr = RES ? residual + row * ldr : nullptr;
  const int nvec = (D + V - 1) / V;
  const int steps = NV ? NV : (nvec + G - 1) / G;
  float keep[kKeep][V];
  float sq = 0.0f;
#pragma unroll kUnroll
  for (int j = 0; j < steps; j++) {
    const int c = (lane + j * G) * V;
    float v[V];
    if (c < D) {
      load_row<T, VECTOR>(xr, c, D, v);
      if constexpr (RES) {
        float r[V];
        load_row<T, VECTOR>(rr, c, D, r);
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = to_f32(from_f32<T>(v[k] + r[k]));  // the rounded residual
        store_row<T, VECTOR>(s_out + row * (int64_t)D, c, D, v);
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) v[k] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < V; k++) sq = __builtin_fmaf(v[k], v[k], sq);
    if constexpr (NV > 0) {
#pragma unroll
      for (int k = 0; k < V; k++) keep[j][k] = v[k];
    }
  }
  sq = group_sum<G>(sq, red);
  const float r = 1.0f / sqrtf(sq / (float)D + eps);
#pragma unroll kUnroll
  for (int j = 0; j < steps; j++) {
    const int c = (lane + j * G) * V;
    float v[V], g[V];
    if constexpr (NV > 0) {
#pragma unroll
      for (int k = 0; k < V; k++) v[k] = keep[j][k];
    } else if (c < D) {  // this lane's own stores above, or the input
      load_row<T, VECTOR>(RES ? s_out + row * (int64_t)D : xr, c, D, v);
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) v[k] = 0.0f;
    }
    if (c < D) {
      load_row<T, VECTOR>(w, c, D, g);
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) g[k] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = v[k] * r * g[k];
    if constexpr (!FP8) {
      if (c < D) store_row<T, VECTOR>(y + row * (int64_t)D, c, D, v);
    } else {
      // 128 columns are the 128 / V lanes from a multiple of 128 / V: their largest magnitude by shuffles (every lane takes part, the
      // ones behind the row's end with zeros).  fmaxf would pass over a NaN: one in the block makes the scale NaN.
      constexpr int L = 128 / V;
      static_assert(G % L == 0, "a block of 128 columns lies within a group");
      float m = 0.0f;
      bool bad = false;
#pragma unroll
      for (int k = 0; k < V; k++) {
        m = fmaxf(m, fabsf(v[k]));
        bad |= v[k] != v[k];
      }
#pragma unroll
      for (int d = 1; d < L; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
      const uint64_t any = __ballot(bad);
      const int first = (threadIdx.x & 63) / L * L;
      const bool nan = ((any >> first) & (L == 64 ? ~0ull : ((1ull << L) - 1))) != 0;
      // 2^-96: a block of zeros (or of values next to nothing) keeps a scale whose reciprocal is finite
      const float scale = nan ? __builtin_nanf("") : fmaxf(m, 0x1p-96f) / 448.0f;
      if (c < D) {
        if (c % 128 == 0) scales[row * (int64_t)((D + 127) / 128) + c / 128] = scale;
        uint32_t pk[V / 4];
#pragma unroll
        for (int k = 0; k < V; k += 4) {
          int u = __builtin_amdgcn_cvt_pk_fp8_f32(v[k] / scale, v[k + 1] / scale, 0, false);
          pk[k / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[k + 2] / scale, v[k + 3] / scale, u, true);
        }
        uint8_t *qr = q + row * (int64_t)D + c;
        if constexpr (VECTOR) {
          if constexpr (V == 8) {
            *reinterpret_cast<dgs_u2 *>(qr) = dgs_u2{pk[0], pk[V / 4 - 1]};
          } else {
            *reinterpret_cast<uint32_t *>(qr) = pk[0];
          }
        } else {
#pragma unroll
          for (int k = 0; k < V; k++)
            if (c + k < D) qr[k] = (uint8_t)(pk[k / 4] >> (8 * (k % 4)));
        }
      }
    }
  }
}

// Backward: workgroup b takes rows b, b + gridDim, ... (a group of G lanes each), keeps its share of dw in registers and leaves it in
// partial[b][D]; rms_norm_dw_kernel sums the partials in a fixed order.  mean(s^2) is taken again from s: it costs no memory access.
template <typename T, bool VECTOR, int G, int NV, bool DS>
__global__ __launch_bounds__(kBlock) void rms_norm_bwd_kernel(int64_t rows, int D, const T *__restrict__ s, const T *__restrict__ w, float eps,
                                                              const T *__restrict__ dy, const T *__restrict__ ds, T *__restrict__ dx,
                                                              float *__restrict__ partial) {
  constexpr int V = kVec<T>;
  constexpr int R = kBlock / G;  // rows in flight in the workgroup
  __shared__ float red[2][2][4];
  __shared__ float join[R > 1 ? (R - 1) * G * NV * V : 1];
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  float g[NV][V], acc[NV][V];
#pragma unroll
  for (int j = 0; j < NV; j++) {
    const int c = (lane + j * G) * V;
    if (c < D) {
      load_row<T, VECTOR>(w, c, D, g[j]);
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) g[j][k] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < V; k++) acc[j][k] = 0.0f;
  }
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * R + sub; row < rows; row += (int64_t)gridDim.x * R, turn ^= 1) {
    const int64_t at = row * (int64_t)D;
    float sv[NV][V], gy[NV][V];
    float sq = 0.0f, dot = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int c = (lane + j * G) * V;
      if (c < D) {
        load_row<T, VECTOR>(s + at, c, D, sv[j]);
        load_row<T, VECTOR>(dy + at, c, D, gy[j]);
      } else {
#pragma unroll
        for (int k = 0; k < V; k++) sv[j][k] = gy[j][k] = 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int k = 0; k < V; k++) {
        sq = __builtin_fmaf(sv[j][k], sv[j][k], sq);
        dot = __builtin_fmaf(sv[j][k] * g[j][k], gy[j][k], dot);
      }
    sq = group_sum<G>(sq, red[turn][0]);  // (two sets of LDS slots: a row's sums are read while the next row's are written)
    dot = group_sum<G>(dot, red[turn][1]);
    const float r = 1.0f / sqrtf(sq / (float)D + eps);
    const float m = r * (dot / (float)D);
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int c = (lane + j * G) * V;
      if (c >= D) continue;
      float o[V];
      if constexpr (DS) {
        load_row<T, VECTOR>(ds + at, c, D, o);
      } else {
#pragma unroll
        for (int k = 0; k < V; k++) o[k] = 0.0f;
      }
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float n = sv[j][k] * r;
        o[k] = __builtin_fmaf(r, __builtin_fmaf(-n, m, g[j][k] * gy[j][k]), o[k]);
        acc[j][k] = __builtin_fmaf(gy[j][k], n, acc[j][k]);
      }
      store_row<T, VECTOR>(dx + at, c, D, o);
    }
  }
  if (!partial) return;
  if constexpr (R > 1) {  // the workgroup's row groups, joined in their order
    if (sub) {
#pragma unroll
      for (int j = 0; j < NV; j++)
#pragma unroll
        for (int k = 0; k < V; k++) join[(((sub - 1) * NV + j) * V + k) * G + lane] = acc[j][k];
    }
    __syncthreads();
    if (sub) return;
    for (int o = 0; o < R - 1; o++)
#pragma unroll
      for (int j = 0; j < NV; j++)
#pragma unroll
        for (int k = 0; k < V; k++) acc[j][k] += join[((o * NV + j) * V + k) * G + lane];
  }
#pragma unroll
  for (int j = 0; j < NV; j++)
#pragma unroll
    for (int k = 0; k < V; k++) {
      const int c = (lane + j * G) * V + k;
      if (c < D) partial[(int64_t)blockIdx.x * D + c] = acc[j][k];
    }
}

// Rows longer than the registers take: three reads of a row from L2 instead of one; dw by columns in a kernel of its own.
template <typename T, bool DS>
__global__ __launch_bounds__(kBlock) void rms_norm_bwd_long_kernel(int D, const T *__restrict__ s, const T *__restrict__ w, float eps,
                                                                   const T *__restrict__ dy, const T *__restrict__ ds, T *__restrict__ dx,
                                                                   float *__restrict__ rstd) {
  __shared__ float red[2][4];
  const int64_t row = blockIdx.x, at = row * (int64_t)D;
  float sq = 0.0f, dot = 0.0f;
  for (int c = threadIdx.x; c < D; c += kBlock) {
    const float v = to_f32(s[at + c]);
    sq = __builtin_fmaf(v, v, sq);
    dot = __builtin_fmaf(v * to_f32(w[c]), to_f32(dy[at + c]), dot);
  }
  sq = group_sum<256>(sq, red[0]);
  dot = group_sum<256>(dot, red[1]);
  const float r = 1.0f / sqrtf(sq / (float)D + eps);
  const float m = r * (dot / (float)D);
  if (rstd && threadIdx.x == 0) rstd[row] = r;
  for (int c = threadIdx.x; c < D; c += kBlock) {
    const float n = to_f32(s[at + c]) * r, o = DS ? to_f32(ds[at + c]) : 0.0f;
    dx[at + c] = from_f32<T>(__builtin_fmaf(r, __builtin_fmaf(-n, m, to_f32(w[c]) * to_f32(dy[at + c])), o));
  }
}
template <typename T>
__global__ __launch_bounds__(kBlock) void rms_norm_dw_long_kernel(int64_t rows, int D, const T *__restrict__ s, const T *__restrict__ dy,
                                                                  const float *__restrict__ rstd, float *__restrict__ partial) {
  const int c = blockIdx.x * kBlock + threadIdx.x;
  if (c >= D) return;
  float acc = 0.0f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y)
    acc = __builtin_fmaf(to_f32(dy[row * (int64_t)D + c]), to_f32(s[row * (int64_t)D + c]) * rstd[row], acc);
  partial[(int64_t)blockIdx.y * D + c] = acc;
}

// dw[c] = sum over the parts, 32 columns x 8 strides of parts a workgroup
template <typename T>
__global__ __launch_bounds__(kBlock) void rms_norm_dw_kernel(int parts, int D, const float *__restrict__ partial, T *__restrict__ dw) {
  __shared__ float sum[8][32];
  const int col = threadIdx.x % 32, sub = threadIdx.x / 32;
  const int c = blockIdx.x * 32 + col;
  float a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
  if (c < D) {
    int p = sub;
    for (; p + 24 < parts; p += 32) {
      a0 += partial[(int64_t)p * D + c];
      a1 += partial[(int64_t)(p + 8) * D + c];
      a2 += partial[(int64_t)(p + 16) * D + c];
      a3 += partial[(int64_t)(p + 24) * D + c];
    }
    for (; p < parts; p += 8) a0 += partial[(int64_t)p * D + c];
  }
  sum[sub][col] = (a0 + a1) + (a2 + a3);
  __syncthreads();
  if (sub == 0 && c < D) {
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) t += sum[k][col];
    dw[c] = from_f32<T>(t);
  }
}

// One group shape for a row of nvec vectors: the smallest that holds it.
//   <= 64 vectors: part of a wave or a wave, one vector a lane; <= 256: a wave, 4 vectors a lane; <= 2048: the workgroup, up to 8.
struct NormShape { int G, NV; };
static NormShape norm_shape(int64_t nvec, int least) {
  if (nvec <= 64) {
    int G = least;
    while (G < nvec) G <<= 1;
    return {G, 1};
  }
  if (nvec <= 128) return {64, 2};
  if (nvec <= 256) return {64, 4};
  if (nvec <= 512) return {256, 2};
  if (nvec <= 1024) return {256, 4};
  if (nvec <= 2048) return {256, 8};
  return {256, 0};
}

template <typename T, bool VECTOR, bool RES, bool FP8>
static int launch_norm(int64_t rows, int D, const T *x, int64_t ldx, const T *res, int64_t ldr, const T *w, float eps, T *y, T *s, uint8_t *q,
                       float *scales, hipStream_t st) {
  const NormShape sh = norm_shape((D + kVec<T> - 1) / kVec<T>, FP8 ? 128 / kVec<T> : 8);
  const int64_t blocks = (rows + kBlock / sh.G - 1) / (kBlock / sh.G);
  if (!grid_ok(blocks)) return DGS_ERANGE;
#define DGS_NORM(G_, NV_)                                                                                                              \
  if (sh.G == G_ && sh.NV == NV_) {                                                                                                    \
    hipLaunchKernelGGL((rms_norm_kernel<T, VECTOR, G_, NV_, RES, FP8>), dim3((unsigned)blocks), dim3(kBlock), 0, st, rows, D, x, ldx, res, ldr, w, \
                       eps, y, s, q, scales);                                                                                          \
    return check_launch();                                                                                                             \
  }
  if constexpr (!FP8) {
    DGS_NORM(8, 1)
  }
  if constexpr (!FP8 || kVec<T> == 8) {
    DGS_NORM(16, 1)
  }
  DGS_NORM(32, 1)
  DGS_NORM(64, 1)
  DGS_NORM(64, 2)
  DGS_NORM(64, 4)
  DGS_NORM(256, 2)
  DGS_NORM(256, 4)
  DGS_NORM(256, 8)
  DGS_NORM(256, 0)
#undef DGS_NORM
  return DGS_EINVAL;
}

template <typename T>
static bool rows_vector(int64_t D, const void *const *ptrs, int np, const int64_t *lds, int nl) {
  if (D % kVec<T>) return false;
  for (int i = 0; i < np; i++)
    if (ptrs[i] && !aligned_to(ptrs[i], 16)) return false;
  for (int i = 0; i < nl; i++)
    if (lds[i] % kVec<T>) return false;
  return true;
}

template <typename T>
static int norm_fwd(int64_t rows, int64_t D, const void *x, int64_t ldx, const void *res, int64_t ldr, const void *w, float eps, void *y, void *s,
                    uint8_t *q, float *scales, hipStream_t st) {
  const void *ptrs[] = {x, res, w, y, s, q};  // (q in 8-byte pieces; 16 is asked of all alike)
  const int64_t lds[] = {ldx, res ? ldr : 0};
  const bool vec = rows_vector<T>(D, ptrs, 6, lds, 2);
  const T *xp = (const T *)x, *rp = (const T *)res, *wp = (const T *)w;
#define DGS_GO(VEC_, RES_, FP8_) \
  return launch_norm<T, VEC_, RES_, FP8_>(rows, (int)D, xp, ldx, rp, ldr, wp, eps, (T *)y, (T *)s, q, scales, st)
  if (q) {
    if (vec) { if (res) DGS_GO(true, true, true); DGS_GO(true, false, true); }
    if (res) DGS_GO(false, true, true);
    DGS_GO(false, false, true);
  }
  if (vec) { if (res) DGS_GO(true, true, false); DGS_GO(true, false, false); }
  if (res) DGS_GO(false, true, false);
  DGS_GO(false, false, false);
#undef DGS_GO
}

// Workgroups of the backward pass: enough to fill the card, few enough that the partial sums of dw stay small beside the rows.
static int64_t bwd_blocks(int64_t rows, int R) {
  const int64_t need = (rows + R - 1) / R;
  return need < 1024 ? need : 1024;
}
constexpr int kLongParts = 64;

template <typename T>
static size_t bwd_ws(int64_t rows, int64_t D) {
  const NormShape sh = norm_shape((D + kVec<T> - 1) / kVec<T>, 8);
  if (sh.NV == 0) return round_up((size_t)rows * 4, 256) + (size_t)kLongParts * D * 4;
  return (size_t)bwd_blocks(rows, kBlock / sh.G) * D * 4;
}

template <typename T>
static int norm_bwd(int64_t rows, int64_t D, const void *s, const void *w, float eps, const void *dy, const void *ds, void *dx, void *dw, char *ws,
                    hipStream_t st) {
  const void *ptrs[] = {s, w, dy, ds, dx};
  const bool vec = rows_vector<T>(D, ptrs, 5, nullptr, 0);
  const NormShape sh = norm_shape((D + kVec<T> - 1) / kVec<T>, 8);
  const T *sp = (const T *)s, *wp = (const T *)w, *dyp = (const T *)dy, *dsp = (const T *)ds;
  float *partial = (float *)ws;
  int64_t parts = 0;
  if (sh.NV == 0) {
    if (!grid_ok(rows)) return DGS_ERANGE;
    float *rstd = (float *)ws;
    partial = (float *)(ws + round_up((size_t)rows * 4, 256));
    if (ds)
      hipLaunchKernelGGL((rms_norm_bwd_long_kernel<T, true>), dim3((unsigned)rows), dim3(kBlock), 0, st, (int)D, sp, wp, eps, dyp, dsp, (T *)dx, dw ? rstd : nullptr);
    else
      hipLaunchKernelGGL((rms_norm_bwd_long_kernel<T, false>), dim3((unsigned)rows), dim3(kBlock), 0, st, (int)D, sp, wp, eps, dyp, dsp, (T *)dx, dw ? rstd : nullptr);
    if (check_launch() != DGS_OK) return DGS_ELAUNCH;
    if (!dw) return DGS_OK;
    parts = rows < kLongParts ? rows : kLongParts;
    hipLaunchKernelGGL((rms_norm_dw_long_kernel<T>), dim3((unsigned)((D + kBlock - 1) / kBlock), (unsigned)parts), dim3(kBlock), 0, st, rows, (int)D, sp, dyp, rstd, partial);
    if (check_launch() != DGS_OK) return DGS_ELAUNCH;
  } else {
    parts = bwd_blocks(rows, kBlock / sh.G);
    float *pp = dw ? partial : nullptr;
#define DGS_BWD(G_, NV_)                                                                                                                       \
  if (sh.G == G_ && sh.NV == NV_) {                                                                                                            \
    if (vec && ds)                                                                                                                             \
      hipLaunchKernelGGL((rms_norm_bwd_kernel<T, true, G_, NV_, true>), dim3((unsigned)parts), dim3(kBlock), 0, st, rows, (int)D, sp, wp, eps, dyp, dsp, (T *)dx, pp);  \
    else if (vec)                                                                                                                              \
      hipLaunchKernelGGL((rms_norm_bwd_kernel<T, true, G_, NV_, false>), dim3((unsigned)parts), dim3(kBlock), 0, st, rows, (int)D, sp, wp, eps, dyp, dsp, (T *)dx, pp); \
    else if (ds)                                                                                                                               \
      hipLaunchKernelGGL((rms_norm_bwd_kernel<T, false, G_, NV_, true>), dim3((unsigned)parts), dim3(kBlock), 0, st, rows, (int)D, sp, wp, eps, dyp, dsp, (T *)dx, pp); \
    else                                                                                                                                       \
      hipLaunchKernelGGL((rms_norm_bwd_kernel<T, false, G_, NV_, false>), dim3((unsigned)parts), dim3(kBlock), 0, st, rows, (int)D, sp, wp, eps, dyp, dsp, (T *)dx, pp); \
  }
    DGS_BWD(8, 1) DGS_BWD(16, 1) DGS_BWD(32, 1) DGS_BWD(64, 1) DGS_BWD(64, 2) DGS_BWD(64, 4) DGS_BWD(256, 2) DGS_BWD(256, 4) DGS_BWD(256, 8)
#undef DGS_BWD
    if (check_launch() != DGS_OK) return DGS_ELAUNCH;
    if (!dw) return DGS_OK;
  }
  hipLaunchKernelGGL((rms_norm_dw_kernel<T>), dim3((unsigned)((D + 31) / 32)), dim3(kBlock), 0, st, (int)parts, (int)D, partial, (T *)dw);
  return check_launch();
}

}  // namespace dgs

using namespace dgs;

static bool norm_sizes_ok(int64_t rows, int64_t D) { return rows <= INT32_MAX && D < INT32_MAX / 64; }

extern "C" int dgs_rms_norm(int dtype, int64_t rows, int64_t D, const void *x, int64_t ldx, const void *residual, int64_t ldr, const void *weight,
                            float eps, void *y, void *s, uint8_t *q, float *scales, dgsStream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || D <= 0 || ldx < 0 || (residual && ldr < 0) || !(eps >= 0.0f)) return DGS_EINVAL;
  if (!norm_sizes_ok(rows, D)) return DGS_ERANGE;
  if (rows == 0) return DGS_OK;
  if (!x || !weight || (residual && !s) || (!residual && s) || (!y == !q) || (!q != !scales)) return DGS_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == DGS_F32) return norm_fwd<float>(rows, D, x, ldx, residual, ldr, weight, eps, y, s, q, scales, st);
  if (dtype == DGS_F16) return norm_fwd<f16>(rows, D, x, ldx, residual, ldr, weight, eps, y, s, q, scales, st);
  return norm_fwd<bf16>(rows, D, x, ldx, residual, ldr, weight, eps, y, s, q, scales, st);
}

extern "C" size_t dgs_rms_norm_bwd_workspace_bytes(int dtype, int64_t rows, int64_t D) {
  if (!dtype_ok(dtype) || rows <= 0 || D <= 0) return 0;
  return dtype == DGS_F32 ? bwd_ws<float>(rows, D) : bwd_ws<f16>(rows, D);
}

extern "C" int dgs_rms_norm_bwd(int dtype, int64_t rows, int64_t D, const void *s, const void *weight, float eps, const void *dy, const void *ds,
                                void *dx, void *dweight, void *workspace, size_t workspace_bytes, dgsStream_t stream) {
  if (!dtype_ok(dtype) || rows <= 0 || D <= 0 || !(eps >= 0.0f)) return DGS_EINVAL;
  if (!norm_sizes_ok(rows, D)) return DGS_ERANGE;
  if (!s || !weight || !dy || !dx) return DGS_EINVAL;
  if (dweight && (!workspace || workspace_bytes < dgs_rms_norm_bwd_workspace_bytes(dtype, rows, D))) return DGS_EWORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  char *ws = static_cast<char *>(workspace);
  if (dtype == DGS_F32) return norm_bwd<float>(rows, D, s, weight, eps, dy, ds, dx, dweight, ws, st);
  if (dtype == DGS_F16) return norm_bwd<f16>(rows, D, s, weight, eps, dy, ds, dx, dweight, ws, st);
  return norm_bwd<bf16>(rows, D, s, weight, eps, dy, ds, dx, dweight, ws, st);
}
