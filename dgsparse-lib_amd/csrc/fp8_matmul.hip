// fp8_matmul.hip -- matrix product of 8-bit floating point (e4m3) operands with a scale for each block of 128, and the quantiser in front of it.
//
//   out[m, n] = sum over blocks b of 128 k:  sa[m, b] sb[n / 128, b]  sum over k in b of a[m, k] b[n, k]
//
// A step of 128 bytes of K is one block: one 16 x 16 x 128 matrix instruction from a zero start gives the inner sum, one multiply-add with
// the two scales' product adds it to the running sum in 32 bits.  The operands' order in the instruction puts m on the lanes, so a lane
// needs one scale of a for each 16 rows; a wave's columns lie within one block of 128, so the scale of b is the wave's.
// Bound: many rows: the matrix cores, with four multiply-adds a lane beside each instruction; few rows: the bytes of b (fp8_few_kernel).
// Measured: 4095 x 11000 x 4096, bf16 out: 196 - 215 us (1.7 - 1.9 PFLOP/s; a large product without block scales, the library's: 2.7);
// 5 x 4096 x 11008: 10.0 us (45 MB: 4.5 TB/s), 1 x 32000 x 4096: 23.4 (5.6).
#include "gemm_core.h"

namespace dgs {

typedef int i32x4 __attribute__((ext_vector_type(4)));
union Slice8 {  // 128 bytes of K for each of 16 rows: per lane the 16 bytes at 16 g and at 64 + 16 g (the same for both operands)
  i32x8 v;
  dgs_u4 u[2];
};
// The sum over a block.  The 8-bit matrix instructions align the 128 products of a sum to the largest and drop what lies some 17 bits below
// it (measured: 1.5e-5 of the result's norm on normal operands, at most 1.2e-4 of the sum of magnitudes on random bit patterns; the older
// 16 x 16 x 32 instruction is no closer).  A result in 16 bits is rounded at 2^-9 or 2^-12 behind that: it takes them, at twice the rate.  A
// result in 32 bits takes the 16-bit instructions, whose sums keep 32 bits; e4m3 values are exact in bf16.
template <typename T>
__device__ __forceinline__ f32x4 block_product(const Slice8 &b, const Slice8 &a) {
  f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (sizeof(T) == 2) {
    // formats 0, 0: e4m3; both hardware scales unused
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.v, a.v, c, 0, 0, 0, 0, 0, 0);
  } else {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    union Wide { bf16x2 p[4]; bf16x8 v; };
#pragma unroll
    for (int k = 0; k < 4; k++) {
      Wide x, y;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        x.p[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b.v[2 * k + h], 1.0f, false);
        x.p[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b.v[2 * k + h], 1.0f, true);
        y.p[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a.v[2 * k + h], 1.0f, false);
        y.p[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a.v[2 * k + h], 1.0f, true);
      }
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, y.v, c, 0, 0, 0);
    }
    return c;
  }
}

struct Scales { const float *a, *b; int64_t blocks; };  // a [M, blocks], b [ceil(N / 128), blocks]

constexpr int kWindow = 8;  // (even: a window's first step is the first of a pair)

template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM *WN) void fp8_kernel(const GemmArgs g, const Scales sc, T *__restrict__ out, float *__restrict__ partial) {
  using G = Gemm<fp8, BM, BN, WM, WN, false, false, kOne>;
  DGS_GEMM_LDS(G)
  static_assert(BN / WN <= 128 && 128 % (BN / WN) == 0, "a wave's columns have one scale");
  const Where at = where_of(g.tiles_m, g.tiles_n);
  const int m0 = at.m * BM, n0 = at.n * BN;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, wm = wave / WN, wn = wave % WN;
  const int steps = (int)sc.blocks, per = (steps + g.splits - 1) / g.splits, s0 = at.z * per, s1 = s0 + per < steps ? s0 + per : steps;
  f32x4 acc[G::FM][G::FN];
#pragma unroll
  for (int i = 0; i < G::FM; i++)
#pragma unroll
    for (int j = 0; j < G::FN; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // The scales for kWindow steps at a time, by way of LDS: the loads take them in rows of kWindow neighbours (a lane's own loads of them
  // would touch 16 lines for each 16 rows: 305 us instead of 221 for 4095 x 11000 x 4096).  Two windows: the next one is loaded in the first
  // step of this one.  Rows behind the matrix are behind the descriptor: 0.
  constexpr int kScaleLoads = BM * kWindow / G::kThreads;
  __shared__ __align__(16) float scales[2][BM * kWindow + 64];  // (behind a's: b's, a row of kWindow for each 128 columns)
  const int64_t scale_bytes = (g.M - m0) * sc.blocks * 4, nb = n0 / 128, b_bytes = ((g.N + 127) / 128 - nb) * sc.blocks * 4;
  const auto sa = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(sc.a + m0 * sc.blocks), 0, scale_bytes < kRange ? (int)scale_bytes : kRange, 0x00027000);
  const auto sb = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(sc.b + nb * sc.blocks), 0, b_bytes < kRange ? (int)b_bytes : kRange, 0x00027000);
  auto load_window = [&](int w) {  // steps s0 + w kWindow ...
    const int s = s0 + w * kWindow + (int)threadIdx.x % kWindow;
#pragma unroll
    for (int q = 0; q < kScaleLoads; q++) {
      const int row = (q * G::kThreads + (int)threadIdx.x) / kWindow;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(sa, (lds_void *)(lds_char *)(&scales[w & 1][(q * G::kWaves + wave) * 64]), 4, s < s1 ? (row * (int)sc.blocks + s) * 4 : (int)kNowhere, 0, 0, 0);
    }
    if (wave == 0) {
      const int row = lane / kWindow;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(sb, (lds_void *)(lds_char *)(&scales[w & 1][BM * kWindow]), 4, s < s1 && row < (BN + 127) / 128 ? (row * (int)sc.blocks + s) * 4 : (int)kNowhere, 0, 0, 0);
    }
  };
  // a step's scales are read from LDS a step ahead
  float f[G::FM], ahead[G::FM], ahead_b = 0.0f;
  auto fetch_scales = [&](int s) {
    const float *p = scales[((s - s0) / kWindow) & 1] + (s - s0) % kWindow;
    ahead_b = p[(BM + ((n0 + wn * (BN / WN)) / 128 - (int)nb)) * kWindow];
#pragma unroll
    for (int i = 0; i < G::FM; i++) ahead[i] = p[(wm * (BM / WM) + (lane & 15) + 16 * i) * kWindow];
  };
  auto take_scales = [&]() {
#pragma unroll
    for (int i = 0; i < G::FM; i++) f[i] = ahead[i] * ahead_b;
  };
  auto compute = [&](const char *la, const char *lb) {
    Slice8 b[G::FN];
#pragma unroll
    for (int j = 0; j < G::FN; j++)
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        Slice s;
        G::TB::read(lb, G::b_row(wn, j), kk, lane, s);
        b[j].u[kk] = s.u;
      }
    Slice8 a[2];  // the next 16 rows' operand is on its way while these are multiplied
    auto fetch = [&](int i) {
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        Slice s;
        G::TA::read(la, wm * (BM / WM) + 16 * i, kk, lane, s);
        a[i & 1].u[kk] = s.u;
      }
    };
    fetch(0);
#pragma unroll
    for (int i = 0; i < G::FM; i++) {
      __builtin_amdgcn_sched_barrier(0);
      if (i + 1 < G::FM) fetch(i + 1);
#pragma unroll
      for (int j = 0; j < G::FN; j++) {
        const f32x4 part = block_product<T>(b[j], a[i & 1]);
#pragma unroll
        for (int k = 0; k < 4; k++) acc[i][j][k] = __builtin_fmaf(part[k], f[i], acc[i][j][k]);
        asm volatile("" : "+v"(acc[i][j]));  // (here, not behind all the products: their sums would fill the registers)
      }
    }
  };
  if (s0 < s1) {
    typename G::Load l;
    G::plan(l, g, m0, n0);
    load_window(0);
    G::load(l, g, m0, n0, s0, steps, 0, ldsA0, ldsB0);
    loads_done();
    fetch_scales(s0);
    int s = s0;
    for (; s + 1 < s1; s += 2) {
      take_scales();
      fetch_scales(s + 1);  // (an odd step of a window: there)
      if ((s - s0) % kWindow == 0 && s + kWindow < s1) load_window((s - s0) / kWindow + 1);
      G::load(l, g, m0, n0, s + 1, steps, 0, ldsA1, ldsB1);
      compute(ldsA0, ldsB0);
      loads_done();
      take_scales();
      if (s + 2 < s1) {
        fetch_scales(s + 2);  // (a new window's first step: loaded since this window's first step)
        G::load(l, g, m0, n0, s + 2, steps, 0, ldsA0, ldsB0);
      }
      compute(ldsA1, ldsB1);
      loads_done();
    }
    take_scales();
    if (s < s1) compute(ldsA0, ldsB0);
  }
#pragma unroll
  for (int i = 0; i < G::FM; i++) {
    const int64_t m = m0 + wm * (BM / WM) + 16 * i + (lane & 15);
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < G::FN; j++) {
      const int64_t n = n0 + G::c_col(wn, j) + 4 * (lane >> 4);
      if (n >= g.N) continue;
      if (partial)
        store4<float>(partial + ((int64_t)at.z * g.M + m) * g.N + n, acc[i][j], g.N - n, g.N % 4 == 0);
      else
        store4<T>(out + m * g.N + n, acc[i][j], g.N - n, g.N % 4 == 0);
    }
  }
}

// Few rows (<= 16 FM): 8 waves share the blocks of K of 16 columns; b goes from memory, whole lines at a time (`turn`), to the matrix instructions.
template <typename T, int FM>
__global__ __launch_bounds__(512) void fp8_few_kernel(const char *__restrict__ a, int64_t lda, const char *__restrict__ b, int64_t ldb, int M, int64_t N, int64_t kbytes,
                                                      const Scales sc, T *__restrict__ out) {
  constexpr int kW = 8;
  __shared__ float sum[kW][16 * FM][17];
  __shared__ __align__(16) char turned[kW][16 * kStepBytes];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, at = (lane >> 4) * 16, piece = (lane & 7) * 16;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const char *pb[2];  // rows 0 - 7 and 8 - 15
#pragma unroll
  for (int q = 0; q < 2; q++) pb[q] = b + (n0 + 8 * q + (lane >> 3) < N ? n0 + 8 * q + (lane >> 3) : N - 1) * ldb + piece;
  const float *sb = sc.b + n0 / 128 * sc.blocks;
  const char *pa[FM];
  const float *sa[FM];
  f32x4 acc[FM];
#pragma unroll
  for (int i = 0; i < FM; i++) {
    const int64_t m = 16 * i + r < M ? 16 * i + r : M - 1;
    pa[i] = a + m * lda + at;
    sa[i] = sc.a + m * sc.blocks;
    acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const dgs_u4 zero = {0u, 0u, 0u, 0u};
  constexpr int U = FM == 1 ? 2 : 1;  // blocks in flight (few: registers for more workgroups on a CU instead; 4 of them: 1 x 32000 x 4096 25.5 us, 2: 23.4)
  for (int64_t k0 = wave; k0 < sc.blocks; k0 += kW * U) {
    Lines y[U];
    Slice8 x[U][FM];
    float f[U][FM];
#pragma unroll
    for (int s = 0; s < U; s++) {
      const int64_t blk = k0 + s * kW;
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        const int64_t k = blk * 128 + kk * 64;
        const bool on = k + at < kbytes;  // (rows are multiples of 16 bytes)
        y[s].u[kk] = blk * 128 + piece < kbytes ? *(const dgs_u4 *)(pb[kk] + blk * 128) : zero;
#pragma unroll
        for (int i = 0; i < FM; i++) x[s][i].u[kk] = on ? *(const dgs_u4 *)(pa[i] + k) : zero;
      }
      const float t = blk < sc.blocks ? sb[blk] : 0.0f;
#pragma unroll
      for (int i = 0; i < FM; i++) f[s][i] = blk < sc.blocks ? sa[i][blk] * t : 0.0f;
    }
#pragma unroll
    for (int s = 0; s < U; s++) {
      Slice t[2];
      turn(turned[wave], lane, y[s], t);
      const Slice8 v = {.u = {t[0].u, t[1].u}};
#pragma unroll
      for (int i = 0; i < FM; i++) {
        const f32x4 part = block_product<T>(v, x[s][i]);
        if (k0 + s * kW < sc.blocks) {
#pragma unroll
          for (int k = 0; k < 4; k++) acc[i][k] = __builtin_fmaf(part[k], f[s][i], acc[i][k]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < FM; i++)
#pragma unroll
    for (int k = 0; k < 4; k++) sum[wave][16 * i + r][4 * (lane >> 4) + k] = acc[i][k];
  __syncthreads();
  for (int e = threadIdx.x; e < 256 * FM; e += 512) {
    const int m = e / 16, c = e % 16;
    if (m >= M || n0 + c >= N) continue;
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < kW; w++) t += sum[w][m][c];
    out[(int64_t)m * N + n0 + c] = from_f32<T>(t);
  }
}

// x in e4m3 with a scale for each ROWS x 128: 32 lanes x 4 columns, 8 rows at a time.  A tile of 128 rows is read twice (the second time
// from L2).  scale = max |x| / 448, at least 2^-96 / 448; a NaN among the values makes it NaN.
template <typename T, int ROWS>
__global__ __launch_bounds__(kBlock) void quantize_kernel(int64_t rows, int64_t cols, const T *__restrict__ x, int64_t ld, bool vec, uint8_t *__restrict__ q,
                                                          float *__restrict__ scales) {
  __shared__ float most[8];
  __shared__ int bad[8];
  const int64_t blocks = (cols + 127) / 128;
  const int sub = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t row, blk;
  if constexpr (ROWS == 1) {
    const int64_t t = (int64_t)blockIdx.x * 8 + sub;
    row = t / blocks;
    blk = t % blocks;
  } else {
    row = (int64_t)blockIdx.x / blocks * ROWS + sub;
    blk = (int64_t)blockIdx.x % blocks;
  }
  const int64_t c = blk * 128 + lane * 4;
  const int64_t end = ROWS == 1 ? (row < rows ? row + 1 : row) : (row - sub + ROWS < rows ? row - sub + ROWS : rows);
  float m = 0.0f;
  int nan = 0;
  for (int64_t r = row; r < end; r += 8) {
    const f32x4 v = c < cols ? load4<T>(x + r * ld + c, cols - c, vec) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      m = fmaxf(m, fabsf(v[k]));
      nan |= v[k] != v[k];
    }
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    m = fmaxf(m, __shfl_xor(m, d, 64));
    nan |= __shfl_xor(nan, d, 64);
  }
  if constexpr (ROWS > 1) {
    if (lane == 0) {
      most[sub] = m;
      bad[sub] = nan;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; k++) {
      m = fmaxf(m, most[k]);
      nan |= bad[k];
    }
  }
  const float scale = nan ? __builtin_nanf("") : fmaxf(m, 0x1p-96f) / 448.0f;
  if (ROWS == 1 ? (lane == 0 && row < rows) : threadIdx.x == 0) scales[ROWS == 1 ? row * blocks + blk : row / ROWS * blocks + blk] = scale;
  if (c >= cols) return;
  for (int64_t r = row; r < end; r += 8) {
    const f32x4 v = load4<T>(x + r * ld + c, cols - c, vec);
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] / scale, v[1] / scale, 0, false);
    u = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] / scale, v[3] / scale, u, true);
    uint8_t *p = q + r * cols + c;
    if (cols % 4 == 0) {
      *reinterpret_cast<int *>(p) = u;
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (c + k < cols) p[k] = (uint8_t)((uint32_t)u >> (8 * k));
    }
  }
}

template <typename T>
static int quantize(int64_t rows, int64_t cols, const void *x, int64_t ld, int block_rows, uint8_t *q, float *scales, hipStream_t st) {
  const bool vec = ld % 4 == 0 && aligned_to(x, 4 * sizeof(T));
  const int64_t blocks = (cols + 127) / 128, grid = block_rows == 1 ? (rows * blocks + 7) / 8 : (rows + 127) / 128 * blocks;
  if (!grid_ok(grid)) return DGS_ERANGE;
  if (block_rows == 1)
    hipLaunchKernelGGL((quantize_kernel<T, 1>), dim3((unsigned)grid), dim3(kBlock), 0, st, rows, cols, (const T *)x, ld, vec, q, scales);
  else
    hipLaunchKernelGGL((quantize_kernel<T, 128>), dim3((unsigned)grid), dim3(kBlock), 0, st, rows, cols, (const T *)x, ld, vec, q, scales);
  return check_launch();
}

// Products that take fp8_few_kernel: beyond 16 rows its reads of a out of L2 for every 16 columns outweigh the 64-row tiles' waste, but for small b
// (few and tiles: 32 x 2048 x 2048 4.9 and 5.9 us, 32 x 4096 x 4096 8.1 and 8.4;  17 x 4096 x 11008 11.2 and 13.2, 32 x 4096 x 11008 15.2 and 13.9, 32 x 32000 x 4096 51
// and 30).
static bool few_rows(int64_t M, int64_t N, int64_t K) { return M <= 16 || (M <= 32 && N * K <= (1 << 24)); }

struct Layout8 {
  bool pad;
  int64_t ldk;
  size_t a, b, partial, total;
  TilePlan plan;
};
static Layout8 layout8(int64_t M, int64_t N, int64_t K, bool wide) {  // wide: the largest tile as well (results in 16 bits)
  Layout8 L;
  size_t at = 0;
  auto take = [&](size_t b) { const size_t o = at; at += round_up(b, 256); return o; };
  L.pad = K % 16 != 0;
  L.ldk = (K + 15) / 16 * 16;
  L.a = take(L.pad ? (size_t)M * L.ldk : 0);
  L.b = take(L.pad ? (size_t)N * L.ldk : 0);
  L.plan = tile_plan(M, N, (K + 127) / 128, 1, false, wide, true);
  L.partial = take(!few_rows(M, N, K) && L.plan.splits > 1 ? (size_t)L.plan.splits * M * N * 4 : 0);
  L.total = at;
  return L;
}

template <typename T>
static int matmul8(int64_t M, int64_t N, int64_t K, const void *a, int64_t lda, const float *sa, const void *b, int64_t ldb, const float *sb, T *out, char *ws, hipStream_t st) {
  const Layout8 L = layout8(M, N, K, sizeof(T) == 2);
  const char *ap = (const char *)a, *bp = (const char *)b;
  if (L.pad) {
    int rc = pad_rows<uint8_t>(M, K, a, lda, L.ldk, ws + L.a, st);
    if (rc == DGS_OK) rc = pad_rows<uint8_t>(N, K, b, ldb, L.ldk, ws + L.b, st);
    if (rc != DGS_OK) return rc;
    ap = ws + L.a;
    bp = ws + L.b;
    lda = ldb = L.ldk;
  }
  const Scales sc = {sa, sb, (K + 127) / 128};
  if (few_rows(M, N, K)) {
    if (!grid_ok((N + 15) / 16, 512)) return DGS_ERANGE;
    const dim3 grid((unsigned)((N + 15) / 16));
    if (M <= 16) hipLaunchKernelGGL((fp8_few_kernel<T, 1>), grid, dim3(512), 0, st, ap, lda, bp, ldb, (int)M, N, L.ldk, sc, out);
    else hipLaunchKernelGGL((fp8_few_kernel<T, 2>), grid, dim3(512), 0, st, ap, lda, bp, ldb, (int)M, N, L.ldk, sc, out);
    return check_launch();
  }
  const TilePlan &p = L.plan;
  float *partial = p.splits > 1 ? (float *)(ws + L.partial) : nullptr;
  const GemmArgs g = {{ap, nullptr}, {bp, nullptr}, lda, ldb, M, N, L.ldk, p.tiles_m, p.tiles_n, p.splits};
  if (!grid_ok((int64_t)p.tiles_m * p.tiles_n, p.shape == kBig ? 512 : 256)) return DGS_ERANGE;
  const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.splits);
  bool done = false;
  if constexpr (sizeof(T) == 2) {
    if (p.shape == kBig) {
      hipLaunchKernelGGL((fp8_kernel<T, 256, 256, 4, 2>), grid, dim3(512), 0, st, g, sc, out, partial);
      done = true;
    }
  }
  if (!done && p.shape == kMid) hipLaunchKernelGGL((fp8_kernel<T, 128, 128, 2, 2>), grid, dim3(256), 0, st, g, sc, out, partial);
  else if (!done) hipLaunchKernelGGL((fp8_kernel<T, 64, 64, 2, 2>), grid, dim3(256), 0, st, g, sc, out, partial);
  if (check_launch() != DGS_OK) return DGS_ELAUNCH;
  if (partial) {
    const int64_t count = M * N;
    hipLaunchKernelGGL((join_splits_kernel<T>), dim3((unsigned)((count + kBlock - 1) / kBlock)), dim3(kBlock), 0, st, count, p.splits, partial, out, out, count);
    return check_launch();
  }
  return DGS_OK;
}

}  // namespace dgs

using namespace dgs;

extern "C" int dgs_quantize_fp8(int dtype, int64_t rows, int64_t cols, const void *x, int64_t ldx, int block_rows, uint8_t *q, float *scales, dgsStream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || cols <= 0 || ldx < 0 || (block_rows != 1 && block_rows != 128)) return DGS_EINVAL;
  if (rows == 0) return DGS_OK;
  if (!x || !q || !scales || (cols % 4 == 0 && !aligned_to(q, 4))) return DGS_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == DGS_F32) return quantize<float>(rows, cols, x, ldx, block_rows, q, scales, st);
  if (dtype == DGS_F16) return quantize<f16>(rows, cols, x, ldx, block_rows, q, scales, st);
  return quantize<bf16>(rows, cols, x, ldx, block_rows, q, scales, st);
}

static bool sizes8_ok(int64_t M, int64_t N, int64_t K) {
  return M < INT32_MAX / 2 && N < INT32_MAX / 2 && K < INT32_MAX / 256 - 64 && ((M + 63) / 64) * ((N + 63) / 64) < INT32_MAX;
}

extern "C" size_t dgs_matmul_fp8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || !sizes8_ok(M, N, K)) return 0;
  const size_t a = layout8(M, N, K, false).total, b = layout8(M, N, K, true).total;  // (the result's type chooses between them)
  return a > b ? a : b;
}

extern "C" int dgs_matmul_fp8_tiles(int out_dtype, int64_t M, int64_t N, int64_t K, int32_t *out) {
  if (!dtype_ok(out_dtype) || M < 0 || N < 0 || K <= 0 || !out) return DGS_EINVAL;
  if (!sizes8_ok(M, N, K)) return DGS_ERANGE;
  const TilePlan p = layout8(M, N, K, out_dtype != DGS_F32).plan;
  out[0] = few_rows(M, N, K) ? 0 : p.shape == kBig ? 256 : p.shape == kMid ? 128 : 64;
  out[1] = p.splits;
  return DGS_OK;
}

extern "C" int dgs_matmul_fp8(int out_dtype, int64_t M, int64_t N, int64_t K, const uint8_t *a, int64_t lda, const float *a_scale, const uint8_t *b, int64_t ldb,
                              const float *b_scale, void *out, void *workspace, size_t workspace_bytes, dgsStream_t stream) {
  if (!dtype_ok(out_dtype) || M < 0 || N < 0 || K <= 0 || lda < 0 || ldb < 0) return DGS_EINVAL;
  if (!sizes8_ok(M, N, K) || lda > INT32_MAX / 256 - 64 || ldb > INT32_MAX / 256 - 64) return DGS_ERANGE;
  if (M == 0 || N == 0) return DGS_OK;
  if (!a || !a_scale || !b || !b_scale || !out || !aligned_to(out, 16)) return DGS_EINVAL;
  // (K a multiple of 16: the operands are read in place, 16 bytes at a time)
  if (K % 16 == 0 && (!aligned_to(a, 16) || !aligned_to(b, 16) || lda % 16 || ldb % 16 || lda < K || ldb < K)) return DGS_EINVAL;
  const size_t need = dgs_matmul_fp8_workspace_bytes(M, N, K);
  if (need && (!workspace || workspace_bytes < need)) return DGS_EWORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  char *ws = static_cast<char *>(workspace);
  if (out_dtype == DGS_F32) return matmul8<float>(M, N, K, a, lda, a_scale, b, ldb, b_scale, (float *)out, ws, st);
  if (out_dtype == DGS_F16) return matmul8<f16>(M, N, K, a, lda, a_scale, b, ldb, b_scale, (f16 *)out, ws, st);
  return matmul8<bf16>(M, N, K, a, lda, a_scale, b, ldb, b_scale, (bf16 *)out, ws, st);
}
