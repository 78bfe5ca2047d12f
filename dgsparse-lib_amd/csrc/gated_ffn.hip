// gated_ffn.hip -- the gated feed-forward product h = act(x Wg^T) * (x Wu^T) in one kernel, with its backward pass.
//
//   forward    g = x Wg^T, u = x Wu^T side by side in one tile (kDual: a wave holds the g and the u of the same columns), h = act(g) u where
//              the tile's sums leave the registers: g and u never reach memory.
//   backward   dg = dh u act'(g), du = dh act(g), rounded once to the type: the operands of the other products.  g and u are those that the
//              forward pass kept (8 bytes for each value of h, one pass over them), or they are made again (4 rows D F flops) and dg, du
//              formed where they leave the registers.
//              dx = dg Wg + du Wu  (one walk over 2 F),  dWg = dg^T x, dWu = du^T x  (sums over the rows, split where there are few tiles).
//
// Bound: the matrix cores (12 rows D F flops forward and backward, 16 with the products made again); for few rows the weights' bytes
// (gated_few_kernel).  Sums are held in 32 bits.
// Measured, forward and backward: 4096 x 4096 x 11008 bf16 2.04 ms (1.09 PFLOP/s; the library's plain products of this shape run at 0.86, of
// 8192^3 at 1.2 - 1.3);  169343 x 128 x 512 fp32 1.18 ms (150 TFLOP/s with the products made again; the library's 32-bit products: 153).
#include "gemm_core.h"

namespace dgs {

// act(g) and act'(g) in 32 bits.  relu;  silu: g s, s (1 + g (1 - s)) with s = 1 / (1 + exp(-g));  gelu: g c, c + g p with the normal
// distribution's c and density p.  c comes from its smaller tail:  c(-|g|) = t P(t) exp(-g^2 / 2), t = 1 / (1 + 0.45 |g| / sqrt(2)), where t P(t)
// is half of exp(y^2) erfc(y), y = |g| / sqrt(2), with P fitted (degree 9, reweighted least squares on Chebyshev points) to 3.2e-8 of it; in 32
// bits c is within 6e-7 of itself for |g| < 4, on either side of 0, and the exponential is the density's too: half the instructions
// of an erf and an exp, beside matrix instructions that it has to keep up with.  v_rcp_f32 is within one unit in the last place.
template <int ACT>
__device__ __forceinline__ float act(float g, float &d) {
  if constexpr (ACT == DGS_ACT_RELU) {
    d = g > 0.0f ? 1.0f : 0.0f;
    return g < 0.0f ? 0.0f : g;  // (a NaN stays)
  } else if constexpr (ACT == DGS_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-g));
    d = s * (1.0f + g * (1.0f - s));
    return g * s;
  } else {
    const float e = __expf(-0.5f * g * g);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.318198051533946386f, fabsf(g), 1.0f));
    float p = -2.074031112e-02f;
    p = __builtin_fmaf(p, t, 9.553859982e-02f);
    p = __builtin_fmaf(p, t, -1.506450521e-01f);
    p = __builtin_fmaf(p, t, 7.154923528e-02f);
    p = __builtin_fmaf(p, t, -1.138132962e-02f);
    p = __builtin_fmaf(p, t, 6.004542311e-02f);
    p = __builtin_fmaf(p, t, 8.761192789e-02f);
    p = __builtin_fmaf(p, t, 1.141373421e-01f);
    p = __builtin_fmaf(p, t, 1.269415080e-01f);
    p = __builtin_fmaf(p, t, 1.269426614e-01f);
    const float q = t * p * e, c = g < 0.0f ? q : 1.0f - q;
    d = __builtin_fmaf(0.39894228040143268f * e, g, c);
    return g * c;
  }
}

// the product of a tile, with its LDS: 16-bit operands straight to LDS, 32-bit ones split on the way
template <typename T, int BM, int BN, int WM, int WN, bool A_KO, bool B_KO, int PAIR>
struct Core {
  using G = Gemm<T, BM, BN, WM, WN, A_KO, B_KO, PAIR>;
  static __device__ __forceinline__ void run(const GemmArgs &g, int m0, int n0, int s0, int s1, int steps, int z, int wm, int wn, int lane, f32x4 (&acc)[G::FM][G::FN]) {
    DGS_GEMM_LDS(G)
    gemm_loop<G>(g, m0, n0, s0, s1, steps, z, ldsA0, ldsB0, ldsA1, ldsB1, wm, wn, lane, acc);
  }
};
template <int BM, int BN, int WM, int WN, bool A_KO, bool B_KO, int PAIR>
struct Core<float, BM, BN, WM, WN, A_KO, B_KO, PAIR> {
  using G = Gemm3<BM, BN, WM, WN, A_KO, B_KO, PAIR>;
  static __device__ __forceinline__ void run(const GemmArgs &g, int m0, int n0, int s0, int s1, int steps, int z, int wm, int wn, int lane, f32x4 (&acc)[G::FM][G::FN]) {
    __shared__ __align__(16) char lds[G::PA::kBytes + G::PB::kBytes];
    G::run(g, m0, n0, s0, s1, steps, z, lds, wm, wn, lane, acc);
  }
};
template <typename T> constexpr int kStepK = kStepBytes / (int)sizeof(T);  // K values a step

struct GatedOut {
  const void *dh;   // backward: [M, F], contiguous
  float *pre;       // forward: where the two products are kept, [2][M, F], or null
  void *o0, *o1;    // forward: h; backward: dg, du
  int64_t F, ldo;   // columns of h / dh; row stride of the outputs (backward: the padded columns F .. ldo are written too, as zeros)
};

template <typename T, int ACT, bool BWD>
__device__ __forceinline__ void gated_store(const GatedOut &o, int64_t M, int64_t m, int64_t n, const f32x4 &g, const f32x4 &u, bool vec) {
  f32x4 a, b;
  if constexpr (BWD) {
    const f32x4 dh = n < o.F ? load4<T>((const T *)o.dh + m * o.F + n, o.F - n, o.F % 4 == 0) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      float d;
      const float v = act<ACT>(g[k], d);
      // (behind F: g = u = 0 and dh = 0 give the zeros that the padding has to hold)
      a[k] = dh[k] * u[k] * d;
      b[k] = dh[k] * v;
    }
    store4<T>((T *)o.o0 + m * o.ldo + n, a, o.ldo - n, true);
    store4<T>((T *)o.o1 + m * o.ldo + n, b, o.ldo - n, true);
  } else {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      float d;
      a[k] = act<ACT>(g[k], d) * u[k];
    }
    store4<T>((T *)o.o0 + m * o.ldo + n, a, o.F - n, vec);
    if (o.pre) {
      store4<float>(o.pre + m * o.F + n, g, o.F - n, vec);
      store4<float>(o.pre + (M + m) * o.F + n, u, o.F - n, vec);
    }
  }
}

// (32 bits: registers for three workgroups on a CU, forward 388 -> 338 us, backward 477 -> 430 of 169343 x 128 x 512; the plain products, which
// read K-outer tiles, would spill at that: 329 -> 410)
template <typename T, int BM, int BN, int WM, int WN, int ACT, bool BWD>
__global__ __launch_bounds__(64 * WM *WN, sizeof(T) == 4 ? 3 : 1) void gated_kernel(const GemmArgs g, const GatedOut o) {
  using G = typename Core<T, BM, BN, WM, WN, false, false, kDual>::G;
  const Where at = where_of(g.tiles_m, g.tiles_n);
  const int m0 = at.m * BM, n0 = at.n * G::kCols;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, wm = wave / WN, wn = wave % WN;
  const int steps = (int)((g.K + kStepK<T> - 1) / kStepK<T>);
  f32x4 acc[G::FM][G::FN];
  Core<T, BM, BN, WM, WN, false, false, kDual>::run(g, m0, n0, 0, steps, steps, 0, wm, wn, lane, acc);
  const bool vec = o.ldo % 4 == 0;
  const int64_t end = BWD ? o.ldo : o.F;
#pragma unroll
  for (int i = 0; i < G::FM; i++) {
    const int64_t m = m0 + wm * (BM / WM) + 16 * i + (lane & 15);
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < G::FN / 2; j++) {
      const int64_t n = n0 + G::c_col(wn, j) + 4 * (lane >> 4);
      if (n < end) gated_store<T, ACT, BWD>(o, g.M, m, n, acc[i][j], acc[i][j + G::FN / 2], vec);
    }
  }
}

// dg and du from kept products: one pass over them and dh.  G lanes a row; the outputs' padding (F .. ldo) gets zeros.
template <typename T, int ACT, bool VECTOR>
__global__ __launch_bounds__(kBlock) void gated_split_kernel(int64_t M, int G, const GatedOut o) {
  constexpr int V = kVec<T>;
  const int lane = threadIdx.x & (G - 1);
  const int64_t m = (int64_t)blockIdx.x * (kBlock / G) + threadIdx.x / G;
  if (m >= M) return;
  const int F = (int)o.F;
  for (int c = lane * V; c < F; c += G * V) {
    float dh[V], a[V], b[V];
    load_row<T, VECTOR>((const T *)o.dh + m * o.F, c, F, dh);
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      const f32x4 g = load4<float>(o.pre + m * o.F + c + q, F - c - q, VECTOR), u = load4<float>(o.pre + (M + m) * o.F + c + q, F - c - q, VECTOR);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        float d;
        const float v = act<ACT>(g[k], d);  // (behind F: dh = 0 and finite others)
        a[q + k] = dh[q + k] * u[k] * d;
        b[q + k] = dh[q + k] * v;
      }
    }
    store_row<T, true>((T *)o.o0 + m * o.ldo, c, F, a);  // (their rows are whole 16-byte pieces)
    store_row<T, true>((T *)o.o1 + m * o.ldo, c, F, b);
  }
}

// Few rows (<= 16 FM): 8 waves share the K of 16 columns of Wg and of Wu, whose rows go from memory, whole lines at a time (`turn`), to the
// matrix instructions; x comes out of L2.  The waves' sums meet in LDS.  3 x 2048 x 5504 fp16: 9.4 us (45 MB: 4.8 TB/s; a plain read of as much, in
// order: 7.1), 1 x 4096 x 11008 bf16: 31.6 us (5.7 TB/s).
template <typename T, int FM, int ACT>
__global__ __launch_bounds__(512, sizeof(T) == 2 && FM < 3 ? 4 : 2) void gated_few_kernel(const char *__restrict__ x, int64_t ldx, const char *__restrict__ wg, const char *__restrict__ wu, int64_t ldw,
                                                        int M, int64_t F, int64_t kbytes, T *__restrict__ h,
                                                        float *__restrict__ pre) {
  constexpr int kW = 8;
  __shared__ float sum[kW][2][16 * FM][17];
  __shared__ __align__(16) char turned[kW][2][16 * kStepBytes];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int r = lane & 15, piece = (lane & 7) * 16;
  const char *pg[2], *pu[2];  // rows 0 - 7 and 8 - 15
#pragma unroll
  for (int q = 0; q < 2; q++) {
    const int64_t n = n0 + 8 * q + (lane >> 3) < F ? n0 + 8 * q + (lane >> 3) : F - 1;
    pg[q] = wg + n * ldw + piece;
    pu[q] = wu + n * ldw + piece;
  }
  const char *px[FM];
#pragma unroll
  for (int i = 0; i < FM; i++) px[i] = x + (int64_t)(16 * i + r < M ? 16 * i + r : M - 1) * ldx + (lane >> 4) * 16;
  f32x4 acc[FM][2];
#pragma unroll
  for (int i = 0; i < FM; i++) acc[i][0] = acc[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const dgs_u4 zero = {0u, 0u, 0u, 0u};
  constexpr int U = FM == 1 ? 4 : 1;  // 128-byte steps in flight (few: registers for more workgroups on a CU instead)
  for (int64_t k0 = wave * 128; k0 < kbytes; k0 += kW * 128 * U) {
    Lines w[U][2];  // (of Wg and of Wu)
    Slice a[U][2][FM];
#pragma unroll
    for (int s = 0; s < U; s++) {
      const int64_t k = k0 + (int64_t)s * kW * 128;
      const bool there = k + piece < kbytes;
#pragma unroll
      for (int q = 0; q < 2; q++) {
        w[s][0].u[q] = there ? *(const dgs_u4 *)(pg[q] + k) : zero;
        w[s][1].u[q] = there ? *(const dgs_u4 *)(pu[q] + k) : zero;
      }
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        const bool on = k + kk * 64 + (lane >> 4) * 16 < kbytes;
#pragma unroll
        for (int i = 0; i < FM; i++) a[s][kk][i].u = on ? *(const dgs_u4 *)(px[i] + k + kk * 64) : zero;
      }
    }
#pragma unroll
    for (int s = 0; s < U; s++) {
      Slice v[2][2], b[2];  // [matrix][kk]
      turn(turned[wave][0], lane, w[s][0], v[0]);
      turn(turned[wave][1], lane, w[s][1], v[1]);
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        b[0] = v[0][kk];
        b[1] = v[1][kk];
        multiply<T>(a[s][kk], b, acc);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < FM; i++)
#pragma unroll
    for (int k = 0; k < 4; k++) {
      sum[wave][0][16 * i + r][4 * (lane >> 4) + k] = acc[i][0][k];
      sum[wave][1][16 * i + r][4 * (lane >> 4) + k] = acc[i][1][k];
    }
  __syncthreads();
  for (int e = threadIdx.x; e < 256 * FM; e += 512) {
    const int m = e / 16, c = e % 16;
    if (m >= M || n0 + c >= F) continue;
    float g = 0.0f, u = 0.0f, d;
#pragma unroll
    for (int w = 0; w < kW; w++) {
      g += sum[w][0][m][c];
      u += sum[w][1][m][c];
    }
    h[(int64_t)m * F + n0 + c] = from_f32<T>(act<ACT>(g, d) * u);
    if (pre) {
      pre[(int64_t)m * F + n0 + c] = g;
      pre[(int64_t)(M + m) * F + n0 + c] = u;
    }
  }
}

// dx and dW: plain products; a split of K leaves its sums in partial[split][matrix][M][N]
struct PlainOut {
  void *C[2];
  int64_t ldc;
  float *partial;
};
template <typename T, int BM, int BN, int WM, int WN, bool A_KO, bool B_KO, int PAIR>
__global__ __launch_bounds__(64 * WM *WN, sizeof(T) == 4 ? 2 : 1) void product_kernel(const GemmArgs g, const PlainOut o) {
  using G = typename Core<T, BM, BN, WM, WN, A_KO, B_KO, PAIR>::G;
  const Where at = where_of(g.tiles_m, g.tiles_n);
  const int z = PAIR == kTwo ? at.z % 2 : 0, split = PAIR == kTwo ? at.z / 2 : at.z;
  const int m0 = at.m * BM, n0 = at.n * BN;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, wm = wave / WN, wn = wave % WN;
  const int steps = (int)((g.K + kStepK<T> - 1) / kStepK<T>), all = PAIR == kSum ? 2 * steps : steps;
  const int per = (all + g.splits - 1) / g.splits, s0 = split * per, s1 = s0 + per < all ? s0 + per : all;
  f32x4 acc[G::FM][G::FN];
  Core<T, BM, BN, WM, WN, A_KO, B_KO, PAIR>::run(g, m0, n0, s0, s1, steps, z, wm, wn, lane, acc);
#pragma unroll
  for (int i = 0; i < G::FM; i++) {
    const int64_t m = m0 + wm * (BM / WM) + 16 * i + (lane & 15);
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < G::FN; j++) {
      const int64_t n = n0 + G::c_col(wn, j) + 4 * (lane >> 4);
      if (n >= g.N) continue;
      if (o.partial) {
        const int64_t mat = (int64_t)split * (PAIR == kTwo ? 2 : 1) + z;
        store4<float>(o.partial + (mat * g.M + m) * g.N + n, acc[i][j], g.N - n, g.N % 4 == 0);
      } else {
        store4<T>((T *)o.C[z] + m * o.ldc + n, acc[i][j], g.N - n, o.ldc % 4 == 0);
      }
    }
  }
}
static bool fits(int64_t M, int64_t N) {  // tiles of the smallest shape in a launch's x dimension
  return ((M + 63) / 64) * ((N + 31) / 32) < INT32_MAX;
}

// The products' tiles.  Forward (backward, made again: cols = the padded F): no split, the activation needs whole sums; 32 bits: no largest tile (three
// planes of 256 + 256 rows leave no room for a second workgroup).
template <typename T>
static TilePlan plan_gated(int64_t rows, int64_t cols, int64_t D) {
  return tile_plan(rows, cols, (D + kStepK<T> - 1) / kStepK<T>, 1, true, sizeof(T) == 2, false);
}
template <typename T>
static TilePlan plan_dx(int64_t rows, int64_t D, int64_t F) {
  return tile_plan(rows, D, 2 * ((F + kStepK<T> - 1) / kStepK<T>), 1, false, sizeof(T) == 2, true);
}
template <typename T>
static TilePlan plan_dw(int64_t rows, int64_t D, int64_t F) {
  return tile_plan(F, D, (rows + kStepK<T> - 1) / kStepK<T>, 2, false, sizeof(T) == 2, true);
}

struct Layout {
  bool pad;          // x and the weights are copied into padded rows
  int64_t ldx, ldg;  // in elements: of x and the weights, and of dg and du
  size_t x, wg, wu, dg, du, partial, total;
};
template <typename T>
static Layout layout(int64_t rows, int64_t D, int64_t F, bool backward, int64_t ldx) {
  Layout L;
  size_t at = 0;
  auto take = [&](size_t b) { const size_t o = at; at += round_up(b, 256); return o; };
  constexpr int V = kVec<T>;
  L.pad = D % V != 0;
  L.ldx = L.pad ? (D + V - 1) / V * V : ldx;
  L.ldg = (F + V - 1) / V * V;
  L.x = take(L.pad ? (size_t)rows * L.ldx * sizeof(T) : 0);
  L.wg = take(L.pad ? (size_t)F * L.ldx * sizeof(T) : 0);
  L.wu = take(L.pad ? (size_t)F * L.ldx * sizeof(T) : 0);
  L.dg = take(backward ? (size_t)rows * L.ldg * sizeof(T) : 0);
  L.du = take(backward ? (size_t)rows * L.ldg * sizeof(T) : 0);
  size_t part = 0;
  if (backward) {
    const TilePlan px = plan_dx<T>(rows, D, F), pw = plan_dw<T>(rows, D, F);
    const size_t bx = px.splits > 1 ? (size_t)px.splits * rows * D * 4 : 0, bw = pw.splits > 1 ? (size_t)pw.splits * 2 * F * D * 4 : 0;
    part = bx > bw ? bx : bw;
  }
  L.partial = take(part);
  L.total = at;
  return L;
}

template <typename T>
struct Operands { const char *x, *wg, *wu; int64_t ldx, ldw; };  // strides in elements
// x and the weights as the 16-byte loads want them
template <typename T>
static int operands(int64_t rows, int64_t D, int64_t F, const void *x, int64_t ldx, const void *wg, const void *wu, int64_t ldw, char *ws, const Layout &L, hipStream_t st,
                    Operands<T> &o) {
  if (!L.pad) {
    if (!rows16(x, D, ldx, sizeof(T)) || !rows16(wg, D, ldw, sizeof(T)) || !rows16(wu, D, ldw, sizeof(T)) || ldx < D || ldw < D) return DGS_EINVAL;
    o = {(const char *)x, (const char *)wg, (const char *)wu, ldx, ldw};
    return DGS_OK;
  }
  int rc = pad_rows<T>(rows, D, x, ldx, L.ldx, ws + L.x, st);
  if (rc == DGS_OK) rc = pad_rows<T>(F, D, wg, ldw, L.ldx, ws + L.wg, st);
  if (rc == DGS_OK) rc = pad_rows<T>(F, D, wu, ldw, L.ldx, ws + L.wu, st);
  o = {ws + L.x, ws + L.wg, ws + L.wu, L.ldx, L.ldx};
  return rc;
}

template <typename T, int ACT, bool BWD>
static int launch_gated(int64_t rows, int64_t D, int64_t F, const Operands<T> &op, const GatedOut &out, hipStream_t st) {
  constexpr bool kWide = sizeof(T) == 2;
  const TilePlan p = plan_gated<T>(rows, BWD ? out.ldo : F, D);
  GemmArgs g = {{op.x, nullptr}, {op.wg, op.wu}, op.ldx * (int64_t)sizeof(T), op.ldw * (int64_t)sizeof(T), rows, F, D, p.tiles_m, p.tiles_n, 1};
  if (!grid_ok((int64_t)p.tiles_m * p.tiles_n, p.shape == kBig ? 512 : 256)) return DGS_ERANGE;
  const dim3 grid((unsigned)(p.tiles_m * p.tiles_n));
  if constexpr (kWide) {
    if (p.shape == kBig) {
      hipLaunchKernelGGL((gated_kernel<T, 256, 256, 2, 4, ACT, BWD>), grid, dim3(512), 0, st, g, out);
      return check_launch();
    }
  }
  if (p.shape == kMid)
    hipLaunchKernelGGL((gated_kernel<T, 128, 128, 2, 2, ACT, BWD>), grid, dim3(256), 0, st, g, out);
  else
    hipLaunchKernelGGL((gated_kernel<T, 64, 64, 2, 2, ACT, BWD>), grid, dim3(256), 0, st, g, out);
  return check_launch();
}
template <typename T, bool A_KO, bool B_KO, int PAIR>
static int launch_product(GemmArgs g, PlainOut o, const TilePlan &p, float *partial, hipStream_t st) {
  constexpr int mats = PAIR == kTwo ? 2 : 1;
  g.tiles_m = p.tiles_m;
  g.tiles_n = p.tiles_n;
  g.splits = p.splits;
  o.partial = p.splits > 1 ? partial : nullptr;
  if (!grid_ok((int64_t)p.tiles_m * p.tiles_n, p.shape == kBig ? 512 : 256)) return DGS_ERANGE;
  const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)(p.splits * mats));
  bool done = false;
  if constexpr (sizeof(T) == 2) {
    if (p.shape == kBig) {
      hipLaunchKernelGGL((product_kernel<T, 256, 256, 2, 4, A_KO, B_KO, PAIR>), grid, dim3(512), 0, st, g, o);
      done = true;
    }
  }
  if (!done && p.shape == kMid)
    hipLaunchKernelGGL((product_kernel<T, 128, 128, 2, 2, A_KO, B_KO, PAIR>), grid, dim3(256), 0, st, g, o);
  else if (!done)
    hipLaunchKernelGGL((product_kernel<T, 64, 64, 2, 2, A_KO, B_KO, PAIR>), grid, dim3(256), 0, st, g, o);
  if (check_launch() != DGS_OK) return DGS_ELAUNCH;
  if (p.splits > 1) {
    const int64_t each = g.M * g.N, count = each * mats;
    hipLaunchKernelGGL((join_splits_kernel<T>), dim3((unsigned)((count + kBlock - 1) / kBlock)), dim3(kBlock), 0, st, count, p.splits, partial, (T *)o.C[0], (T *)o.C[1], each);
    return check_launch();
  }
  return DGS_OK;
}

// Products that take gated_few_kernel.  Beyond 48 rows its reads of x out of L2 for every 16 columns cost more than the 64-row tiles' waste, if
// those fill the card and the weights are in its last cache.  Few and tiles, us, called again on the same weights: 2048 x 5504 fp16: 32 rows 13.9 and
// 18.5, 48 rows 17.7 and 18.6, 64 rows 22.1 and 18.8;  64 x 4096 x 4096 bf16 (128 tiles) 20.9 and 33.7;  1024 x 4096 fp32: 48 rows 15.1 and 22.9, 64 rows 19.3 and
// 23.0.  On weights that come from memory, 64 rows, bf16: 4096 x 2048 24.9 and 50.8, 4096 x 4096 27.1 and 52.6, 4096 x 5504 47.2 and 52.3, 4096 x 8192 49.3 and
// 52.9, 2048 x 4096 17.2 and 27.4, 2048 x 5504 27.4 and 28.4.
template <typename T>
static bool few_rows(int64_t rows, int64_t F) {
  return rows <= 48 || (rows <= 64 && (sizeof(T) == 4 || (F + 31) / 32 < cu_count() * 5 / 8));
}

template <typename T, int ACT>
static int ffn_fwd(int64_t rows, int64_t D, int64_t F, const void *x, int64_t ldx, const void *wg, const void *wu, int64_t ldw, void *h, float *pre, char *ws, hipStream_t st) {
  const Layout L = layout<T>(rows, D, F, false, ldx);
  Operands<T> op;
  const int rc = operands<T>(rows, D, F, x, ldx, wg, wu, ldw, ws, L, st, op);
  if (rc != DGS_OK) return rc;
  if (few_rows<T>(rows, F)) {
    if (!grid_ok((F + 15) / 16, 512)) return DGS_ERANGE;
    const dim3 grid((unsigned)((F + 15) / 16));
    const int64_t kb = (int64_t)(L.pad ? L.ldx : D) * (int64_t)sizeof(T), lx = op.ldx * (int64_t)sizeof(T), lw = op.ldw * (int64_t)sizeof(T);
#define DGS_FEW(FM_) hipLaunchKernelGGL((gated_few_kernel<T, FM_, ACT>), grid, dim3(512), 0, st, op.x, lx, op.wg, op.wu, lw, (int)rows, F, kb, (T *)h, pre)
    if (rows <= 16) DGS_FEW(1);
    else if (rows <= 32) DGS_FEW(2);
    else if (rows <= 48) DGS_FEW(3);
    else DGS_FEW(4);
#undef DGS_FEW
    return check_launch();
  }
  const GatedOut out = {nullptr, pre, h, nullptr, F, F};
  return launch_gated<T, ACT, false>(rows, D, F, op, out, st);
}

template <typename T, int ACT>
static int ffn_bwd(int64_t rows, int64_t D, int64_t F, const void *x, int64_t ldx, const void *wg, const void *wu, int64_t ldw, const float *pre, const void *dh, void *dx, void *dwg,
                   void *dwu, char *ws, hipStream_t st) {
  const Layout L = layout<T>(rows, D, F, true, ldx);
  Operands<T> op;
  int rc = operands<T>(rows, D, F, x, ldx, wg, wu, ldw, ws, L, st, op);
  if (rc != DGS_OK) return rc;
  constexpr int64_t size = sizeof(T);
  char *dg = ws + L.dg, *du = ws + L.du;
  const GatedOut out = {dh, const_cast<float *>(pre), dg, du, F, L.ldg};
  if (pre) {
    int G = 1;
    while (G < kBlock && G * kVec<T> < F) G <<= 1;
    const int64_t blocks = (rows + kBlock / G - 1) / (kBlock / G);
    if (!grid_ok(blocks)) return DGS_ERANGE;
    const dim3 grid((unsigned)blocks);
    if (F % kVec<T> == 0)
      hipLaunchKernelGGL((gated_split_kernel<T, ACT, true>), grid, dim3(kBlock), 0, st, rows, G, out);
    else
      hipLaunchKernelGGL((gated_split_kernel<T, ACT, false>), grid, dim3(kBlock), 0, st, rows, G, out);
    rc = check_launch();
  } else {
    rc = launch_gated<T, ACT, true>(rows, D, F, op, out, st);
  }
  float *partial = (float *)(ws + L.partial);
  if (rc == DGS_OK && dx) {  // dx [rows, D] = dg Wg + du Wu: K = F, the weights K-outer
    GemmArgs g = {{dg, du}, {op.wg, op.wu}, L.ldg * size, op.ldw * size, rows, D, F, 0, 0, 1};
    PlainOut o = {{dx, nullptr}, D, nullptr};
    rc = launch_product<T, false, true, kSum>(g, o, plan_dx<T>(rows, D, F), partial, st);
  }
  if (rc == DGS_OK && dwg) {  // dWg, dWu [F, D] = dg^T x, du^T x: K = rows, both operands K-outer
    GemmArgs g = {{dg, du}, {op.x, nullptr}, L.ldg * size, op.ldx * size, F, D, rows, 0, 0, 1};
    PlainOut o = {{dwg, dwu}, D, nullptr};
    rc = launch_product<T, true, true, kTwo>(g, o, plan_dw<T>(rows, D, F), partial, st);
  }
  return rc;
}

static int edge(Shape s) { return s == kBig ? 256 : s == kMid ? 128 : 64; }
template <typename T>
static void tiles(int64_t rows, int64_t D, int64_t F, int32_t *out) {
  const TilePlan p[] = {plan_gated<T>(rows, F, D), plan_dx<T>(rows, D, F), plan_dw<T>(rows, D, F)};
  for (int i = 0; i < 3; i++) {
    out[2 * i] = edge(p[i].shape);
    out[2 * i + 1] = p[i].splits;
  }
  if (few_rows<T>(rows, F)) out[0] = 0;
}

}  // namespace dgs

using namespace dgs;

static int ffn_sizes(int dtype, int activation, int64_t rows, int64_t D, int64_t F, int64_t ldx, int64_t ldw) {
  if (!dtype_ok(dtype) || activation < DGS_ACT_SILU || activation > DGS_ACT_RELU || rows < 0 || D <= 0 || F <= 0 || ldx < 0 || ldw < 0) return DGS_EINVAL;
  const int64_t size = (int64_t)dtype_bytes(dtype);
  // offsets within a tile are 32 bits wide: 256 rows of any operand
  const int64_t most = INT32_MAX / 256 / size - 64;
  if (rows > INT32_MAX / 2 || D > most || F > most || ldx > most || ldw > most || !fits(rows, F) || !fits(rows, D) || !fits(F, D)) return DGS_ERANGE;
  return DGS_OK;
}

extern "C" size_t dgs_gated_ffn_workspace_bytes(int dtype, int64_t rows, int64_t D, int64_t F, int backward) {
  if (!dtype_ok(dtype) || rows <= 0 || D <= 0 || F <= 0) return 0;
  return dtype == DGS_F32 ? layout<float>(rows, D, F, backward, D).total : layout<f16>(rows, D, F, backward, D).total;
}

extern "C" int dgs_gated_ffn_tiles(int dtype, int64_t rows, int64_t D, int64_t F, int32_t *out) {
  const int rc = ffn_sizes(dtype, DGS_ACT_SILU, rows, D, F, 0, 0);
  if (rc != DGS_OK) return rc;
  if (!out) return DGS_EINVAL;
  if (dtype == DGS_F32) tiles<float>(rows, D, F, out);
  else tiles<f16>(rows, D, F, out);
  return DGS_OK;
}

#define DGS_ACTS(T, CALL)                                      \
  switch (activation) {                                        \
    case DGS_ACT_SILU: return CALL<T, DGS_ACT_SILU> ARGS;      \
    case DGS_ACT_GELU: return CALL<T, DGS_ACT_GELU> ARGS;      \
    default: return CALL<T, DGS_ACT_RELU> ARGS;                \
  }

extern "C" int dgs_gated_ffn(int dtype, int activation, int64_t rows, int64_t D, int64_t F, const void *x, int64_t ldx, const void *w_gate, const void *w_up, int64_t ldw,
                             void *h, float *pre, void *workspace, size_t workspace_bytes, dgsStream_t stream) {
  const int rc = ffn_sizes(dtype, activation, rows, D, F, ldx, ldw);
  if (rc != DGS_OK) return rc;
  if (rows == 0) return DGS_OK;
  if (!x || !w_gate || !w_up || !h || !aligned_to(h, 16) || !aligned_to(pre, 16)) return DGS_EINVAL;
  const size_t need = dgs_gated_ffn_workspace_bytes(dtype, rows, D, F, 0);
  if (need && (!workspace || workspace_bytes < need)) return DGS_EWORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  char *ws = static_cast<char *>(workspace);
#define ARGS (rows, D, F, x, ldx, w_gate, w_up, ldw, h, pre, ws, st)
  if (dtype == DGS_F32) DGS_ACTS(float, ffn_fwd)
  if (dtype == DGS_F16) DGS_ACTS(f16, ffn_fwd)
  DGS_ACTS(bf16, ffn_fwd)
#undef ARGS
}

extern "C" int dgs_gated_ffn_bwd(int dtype, int activation, int64_t rows, int64_t D, int64_t F, const void *x, int64_t ldx, const void *w_gate, const void *w_up, int64_t ldw,
                                 const float *pre, const void *dh, void *dx, void *dw_gate, void *dw_up, void *workspace, size_t workspace_bytes, dgsStream_t stream) {
  const int rc = ffn_sizes(dtype, activation, rows, D, F, ldx, ldw);
  if (rc != DGS_OK) return rc;
  if (rows == 0 || !x || !w_gate || !w_up || !dh || !dw_gate != !dw_up || !aligned_to(dh, 16) || !aligned_to(dx, 16) || !aligned_to(dw_gate, 16) || !aligned_to(dw_up, 16) || !aligned_to(pre, 16))
    return DGS_EINVAL;
  const size_t need = dgs_gated_ffn_workspace_bytes(dtype, rows, D, F, 1);
  if (!workspace || workspace_bytes < need) return DGS_EWORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  char *ws = static_cast<char *>(workspace);
#define ARGS (rows, D, F, x, ldx, w_gate, w_up, ldw, pre, dh, dx, dw_gate, dw_up, ws, st)
  if (dtype == DGS_F32) DGS_ACTS(float, ffn_bwd)
  if (dtype == DGS_F16) DGS_ACTS(f16, ffn_bwd)
  DGS_ACTS(bf16, ffn_bwd)
#undef ARGS
}
