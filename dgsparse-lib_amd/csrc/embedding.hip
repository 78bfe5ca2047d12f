// embedding.hip -- embedding lookup with scaling, and the table's gradient by sorted tokens.
//
//   out[p, :] = scale * table[ids[p], :]              a negative id is "no token": a row of zeros; an id >= V gives a row of NaN (nothing is
//                                                     read out of bounds, and the mistake is seen)
//   dtable[v, :] = scale * sum over p with ids[p] = v of dout[p, :], in a fixed order         (ids that are negative, >= V or equal to the
//                                                     padding id add to no row; a row without a token is 0)
//
// Lookup: HBM-bound gather, each row read once in 16-byte pieces.
// Gradient: positions are sorted by id with the position as the tie-break (embedding_rank / count / place), so every row's sum has one fixed order
// and no atomics.  The sorted list is cut into chunks of 32 or 64 positions; a group of lanes walks a chunk with a running sum in 32 bits
// and writes each row that lies within its chunk.  A row whose positions cross a chunk's border (a frequent token) leaves partial sums in the
// workspace, which embedding_join adds up in chunk order.  Rows without a token are cleared by workgroups of the same launch: they find
// the few ids of their share of the table by binary search in the sorted list, so the table is written once and read never.
// Measured (kernel time): 16384 tokens of 131072 x 4096 bf16: lookup 50 us (5.4 TB/s), sort 28 (two passes of two launches), gradient 221
// (1.07 GB written, 0.13 read: 5.5 TB/s), join 12;  100003 nodes of 169343 x 128 fp32: 21, 29, 45 (3.1 TB/s), 6.
#include "dense_common.h"

namespace dgs {

constexpr int kSortSmall = 8192;   // positions up to here: one launch that counts ranks (n^2 comparisons; at 8192 either sort makes 53 us with an 87 MB gradient behind it, at 4000 this one 42)
constexpr int kSortWaves = 8;      // waves of a radix-sort workgroup
constexpr int kSortBits = 9;       // at most this many bits a pass (512 bins)
constexpr int kSortBlocks = 256;   // at most this many workgroups a pass (each reads all the others' counts)

template <typename I>
__device__ __forceinline__ uint32_t token_key(I id, int64_t V, int64_t pad) {
  const int64_t v = (int64_t)id;
  return v < 0 || v >= V || v == pad ? (uint32_t)V : (uint32_t)v;  // V: adds to no row, sorted behind all others
}

// ---- lookup ----------------------------------------------------------------------------------------------------------------
// G lanes a row (a power of two <= 256), kBlock / G rows a workgroup.
template <typename T, typename I, bool VECTOR>
__global__ __launch_bounds__(kBlock) void embedding_fwd_kernel(int64_t n, int64_t V, int D, int G, const I *__restrict__ ids,
                                                               const T *__restrict__ table, int64_t ld, float scale, T *__restrict__ out) {
  constexpr int W = kVec<T>;
  const int lane = threadIdx.x & (G - 1);
  const int64_t p = (int64_t)blockIdx.x * (kBlock / G) + threadIdx.x / G;
  if (p >= n) return;
  const int64_t id = (int64_t)ids[p];
  const bool there = id >= 0 && id < V;
  const T *row = table + (there ? id : 0) * ld;
  const float none = id < 0 ? 0.0f : __builtin_nanf("");
  for (int c = lane * W; c < D; c += G * W) {
    float x[W];
    if (there) {
      load_row<T, VECTOR>(row, c, D, x);
#pragma unroll
      for (int k = 0; k < W; k++) x[k] *= scale;
    } else {
#pragma unroll
      for (int k = 0; k < W; k++) x[k] = none;
    }
    store_row<T, VECTOR>(out + p * (int64_t)D, c, D, x);
  }
}

// ---- sorting ---------------------------------------------------------------------------------------------------------------
// Few positions: the place of (key, p) in the sorted list is the number of pairs in front of it.  A workgroup ranks 16 positions, 16
// threads each a sixteenth of the list out of LDS, four keys a read; no pass waits for another.
template <typename I>
__global__ __launch_bounds__(kBlock) void embedding_rank_kernel(int n, int64_t V, int64_t pad, const I *__restrict__ ids,
                                                                uint32_t *__restrict__ skey, int *__restrict__ spos) {
  __shared__ __align__(16) uint32_t key[kSortSmall];
  __shared__ int part[16][16];
  const int n4 = (n + 3) / 4;
  for (int p = threadIdx.x; p < 4 * n4; p += kBlock) key[p] = p < n ? token_key(ids[p], V, pad) : 0xffffffffu;  // (behind the list: behind every pair)
  __syncthreads();
  const int mine = threadIdx.x & 15, sub = threadIdx.x >> 4;
  const int p = blockIdx.x * 16 + mine;
  const uint32_t k = p < n ? key[p] : 0u;
  const int len = (n4 + 15) / 16, lo = sub * len, hi = lo + len < n4 ? lo + len : n4;
  int before = 0;
#pragma unroll 4
  for (int o = lo; o < hi; o++) {
    const dgs_u4 v = *reinterpret_cast<const dgs_u4 *>(&key[4 * o]);
#pragma unroll
    for (int j = 0; j < 4; j++) before += (v[j] < k) | ((v[j] == k) & (4 * o + j < p));
  }
  part[sub][mine] = before;
  __syncthreads();
  if (sub == 0 && p < n) {
    int at = 0;
#pragma unroll
    for (int s = 0; s < 16; s++) at += part[s][mine];
    skey[at] = k;
    spos[at] = p;
  }
}

// Many positions: a stable radix sort from the low digit, `tile` positions a workgroup, two launches a pass: counts, then placement.  (Counting
// the next digit while placing saves a launch and loses more to the adds that meet on a frequent token's counter: 77 -> 86 us for
// 100003 positions of a Zipf law with the gradient behind it.)
template <typename I>
__global__ __launch_bounds__(kSortWaves *kWave) void embedding_count_kernel(int64_t n, int64_t V, int64_t pad, int tile, int shift, int bits,
                                                                            const I *__restrict__ ids, const uint32_t *__restrict__ kin, int *__restrict__ hist) {
  __shared__ int cnt[1 << kSortBits];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += blockDim.x) cnt[b] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * tile, hi = lo + tile < n ? lo + tile : n;
  for (int64_t p = lo + threadIdx.x; p < hi; p += blockDim.x) {
    const uint32_t k = kin ? kin[p] : token_key(ids[p], V, pad);
    atomicAdd(&cnt[(k >> shift) & (bins - 1)], 1);  // (a count: its order changes nothing)
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += blockDim.x) hist[(int64_t)blockIdx.x * bins + b] = cnt[b];
}

template <typename I>
__global__ __launch_bounds__(kSortWaves *kWave) void embedding_place_kernel(int64_t n, int64_t V, int64_t pad, int tile, int shift, int bits,
                                                                            const I *__restrict__ ids, const uint32_t *__restrict__ kin,
                                                                            const int *__restrict__ pin, const int *__restrict__ hist,
                                                                            uint32_t *__restrict__ kout, int *__restrict__ pout) {
  __shared__ int off[kSortWaves][1 << kSortBits];  // next place of a digit for each wave's part of the tile
  __shared__ int wsum[kSortWaves];
  static_assert((1 << kSortBits) <= kSortWaves * kWave, "a thread for each bin");
  const int bins = 1 << bits, t = threadIdx.x, wave = t / kWave, lane = t % kWave;
  const int64_t lo = (int64_t)blockIdx.x * tile, hi = lo + tile < n ? lo + tile : n;
  const int share = tile / kSortWaves;  // (a multiple of 64)
  const int64_t wlo = lo + (int64_t)wave * share, whi = wlo + share < hi ? wlo + share : hi;
  for (int b = t; b < kSortWaves << kSortBits; b += blockDim.x) off[b >> kSortBits][b & ((1 << kSortBits) - 1)] = 0;
  __syncthreads();
  for (int64_t p = wlo + lane; p < whi; p += kWave) {
    const uint32_t k = kin ? kin[p] : token_key(ids[p], V, pad);
    atomicAdd(&off[wave][(k >> shift) & (bins - 1)], 1);
  }
  // this thread's digit: positions with it in all workgroups, and in those in front of this one
  int all = 0, front = 0;
  if (t < bins) {
#pragma unroll 32
    for (int b = 0; b < (int)gridDim.x; b++) {  // (independent reads out of L2: as many as registers take are in flight)
      const int h = hist[(int64_t)b * bins + t];
      all += h;
      front += b < (int)blockIdx.x ? h : 0;
    }
  }
  int scan = all;  // inclusive over the digits: in the wave, then over the waves
  for (int d = 1; d < kWave; d <<= 1) {
    const int o = __shfl_up(scan, d, 64);
    if (lane >= d) scan += o;
  }
  if (lane == kWave - 1) wsum[wave] = scan;
  __syncthreads();
  if (t < bins) {
    int base = scan - all + front;
    for (int w = 0; w < wave; w++) base += wsum[w];
    for (int w = 0; w < kSortWaves; w++) {  // the waves' parts follow each other
      const int c = off[w][t];
      off[w][t] = base;
      base += c;
    }
  }
  __syncthreads();
  // placement: each wave goes through its part 64 positions at a time; lanes with the same digit rank among themselves by ballots.  Only
  // this wave touches off[wave]; its LDS accesses are kept in program order by the wave barriers.
  for (int64_t p0 = wlo; p0 < whi; p0 += kWave) {
    const int64_t p = p0 + lane;
    const bool on = p < whi;
    const uint32_t k = on ? (kin ? kin[p] : token_key(ids[p], V, pad)) : 0u;
    const int digit = (int)((k >> shift) & (bins - 1));
    uint64_t peers = __ballot(on);
    for (int b = 0; b < bits; b++) {
      const uint64_t set = __ballot((digit >> b) & 1);
      peers &= (digit >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(peers & ((1ull << lane) - 1));
    int at = 0;
    if (on) at = off[wave][digit] + rank;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (on && rank == 0) off[wave][digit] = at + __popcll(peers);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (on) {
      kout[at] = k;
      pout[at] = pin ? pin[p] : (int)p;
    }
  }
}

// ---- gradient --------------------------------------------------------------------------------------------------------------
// Where the first key >= `key` stands in the sorted list skey[0, n) of every `stride`-th key: a wave splits the range 64-fold, 3 steps for
// 2^18 positions.  Every lane of the wave gets the answer in [0, n].
__device__ __forceinline__ int64_t lower_bound_wave(const uint32_t *__restrict__ skey, int64_t stride, int64_t n, uint32_t key) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, hi = n;
  while (hi > lo) {
    const int64_t step = (hi - lo + kWave - 1) / kWave, at = lo + lane * step;
    // probes in front of the answer: the first `less` lanes
    const int less = __popcll(__ballot(at < hi && skey[(at < hi ? at : lo) * stride] < key));
    const int64_t nlo = less ? lo + (int64_t)(less - 1) * step + 1 : lo, nhi = lo + (int64_t)less * step;
    hi = nhi < hi ? nhi : hi;
    lo = nlo;
  }
  return lo;
}

constexpr int kLeastLanes = 8;                 // of a group
constexpr int kHeld = kBlock / kLeastLanes * 64;  // positions of a workgroup, at most

// Workgroups [0, work): chunks of the sorted list, kBlock / G of them each, `tiles` workgroups for the columns.  Behind them: rows without a
// token, which stream to memory while the chunks wait for theirs.  Partial rows: slot 2c for the row that chunk c goes on with from the
// chunk before, slot 2c + 1 for the row that starts in chunk c and goes on behind it.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(kBlock) void embedding_bwd_kernel(int64_t n, int64_t V, int D, int G, int chunk, int64_t n_chunks, int tiles, int64_t work, int fill_rows, int keep,
                                                               const uint32_t *__restrict__ skey, const int *__restrict__ spos,
                                                               const T *__restrict__ dout, int64_t ldo, float scale, T *__restrict__ dtable,
                                                               float *__restrict__ partial) {
  constexpr int W = kVec<T>;
  const int t = threadIdx.x, lane = t & (G - 1);
  if ((int64_t)blockIdx.x >= work) {
    // fill_rows (<= 256) rows from v0; the sorted list's part with these ids lies between two lower bounds
    __shared__ uint32_t seen[8];
    __shared__ int64_t bound[2];
    const int64_t v0 = ((int64_t)blockIdx.x - work) * fill_rows, v1 = v0 + fill_rows < V ? v0 + fill_rows : V;
    if (t < 8) seen[t] = 0u;
    if (t < 2 * kWave) {
      const int64_t at = lower_bound_wave(skey, 1, n, (uint32_t)(t < kWave ? v0 : v1));
      if ((t & 63) == 0) bound[t / kWave] = at;
    }
    __syncthreads();
    for (int64_t q = bound[0] + t; q < bound[1]; q += kBlock) {
      const int r = (int)((int64_t)skey[q] - v0);
      atomicOr(&seen[r >> 5], 1u << (r & 31));
    }
    __syncthreads();
    float zero[W];
#pragma unroll
    for (int k = 0; k < W; k++) zero[k] = 0.0f;
    for (int64_t v = v0 + t / G; v < v1; v += kBlock / G) {
      const int r = (int)(v - v0);
      if ((seen[r >> 5] >> (r & 31)) & 1) continue;
      if (keep) {
        for (int c = lane * W; c < D; c += G * W) store_row<T, VECTOR>(dtable + v * (int64_t)D, c, D, zero);
      } else {
        for (int c = lane * W; c < D; c += G * W) store_row_stream<T, VECTOR>(dtable + v * (int64_t)D, c, D, zero);
      }
    }
    return;
  }
  // the workgroup's keys (with one neighbour at either end) and positions, read once
  __shared__ uint32_t key[kHeld + 2];
  __shared__ int pos[kHeld];
  const int64_t wb = (int64_t)blockIdx.x / tiles, p0 = wb * (kBlock / G) * chunk;
  const int held = (int)(n - p0 < (int64_t)(kBlock / G) * chunk ? n - p0 : (int64_t)(kBlock / G) * chunk);
  for (int i = t; i < held + 2; i += kBlock) {
    const int64_t q = p0 + i - 1;
    key[i] = q >= 0 && q < n ? skey[q] : 0xffffffffu;  // (no key: keys are at most V)
    if (i < held) pos[i] = spos[p0 + i];
  }
  __syncthreads();
  const int64_t ch = wb * (kBlock / G) + t / G;
  const int c = ((int)((int64_t)blockIdx.x % tiles) * G + lane) * W;
  if (ch >= n_chunks || c >= D) return;
  const int q0 = t / G * chunk, q1 = q0 + chunk < held ? q0 + chunk : held;
  bool head = key[q0] == key[q0 + 1];  // the first row goes on from the chunk before
  float acc[W];
#pragma unroll
  for (int k = 0; k < W; k++) acc[k] = 0.0f;
  constexpr int U = 8;  // rows in flight
  for (int q = q0; q < q1; q += U) {
    float x[U][W];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int at = q + u < q1 ? q + u : q1 - 1;
      if (key[at + 1] < (uint32_t)V) load_row<T, VECTOR>(dout + (int64_t)pos[at] * ldo, c, D, x[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint32_t now = key[(q + u < q1 ? q + u : q1 - 1) + 1];
      if (q + u >= q1 || now >= (uint32_t)V) break;  // (ids that add to no row come last)
#pragma unroll
      for (int k = 0; k < W; k++) acc[k] += x[u][k];
      const bool on = key[q + u + 2] == now;  // the row goes on behind this position
      if (on && q + u + 1 < q1) continue;
      if (head || on) {
        float *slot = partial + (2 * ch + (head ? 0 : 1)) * (int64_t)D;
#pragma unroll
        for (int k = 0; k < W; k++)
          if (c + k < D) slot[c + k] = acc[k];
      } else {
#pragma unroll
        for (int k = 0; k < W; k++) acc[k] *= scale;
        store_row<T, VECTOR>(dtable + (int64_t)now * D, c, D, acc);
      }
      head = false;
#pragma unroll
      for (int k = 0; k < W; k++) acc[k] = 0.0f;
    }
  }
}

// Border b between chunks b - 1 and b: the workgroups of the row that starts in chunk b - 1 and goes on in chunk b add up its partial
// sums: the start's, then one of each chunk up to the last.  32 columns x 8 shares of the chunks; the shares' sums are joined in order.
template <typename T, int V>  // V columns a lane: 4, or 1 where a row of partial sums is no multiple of 16 bytes
__global__ __launch_bounds__(kBlock) void embedding_join_kernel(int64_t first, int64_t vocab, int D, int chunk, int64_t n_chunks, const uint32_t *__restrict__ skey,
                                                                float scale, const float *__restrict__ partial, T *__restrict__ dtable) {
  const int64_t b = first + blockIdx.x;
  const int64_t at = b * chunk;
  const uint32_t key = skey[at];
  const uint32_t prev = skey[at - 1], start = b > 1 ? skey[at - chunk - 1] : 0xffffffffu;
  if (key >= (uint32_t)vocab || prev != key || start == key) return;  // (start == key: an earlier border owns the row)
  __shared__ int64_t end;
  __shared__ __align__(16) float sum[8][32 * V];
  if (threadIdx.x < kWave) {  // the last chunk that begins within the row, by the chunks' first keys
    const int64_t behind = b + lower_bound_wave(skey + at, chunk, n_chunks - b, key + 1);
    if (threadIdx.x == 0) end = behind - 1;
  }
  __syncthreads();
  const int col = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const int64_t m = end - b + 1, len = (m + 7) / 8;  // chunks b .. end, an eighth each
  const int64_t lo = b + sub * len, hi = lo + len < end + 1 ? lo + len : end + 1;
  for (int c0 = (int)blockIdx.y * 32 * V; c0 < D; c0 += (int)gridDim.y * 32 * V) {
    const int c = c0 + col * V;
    float a[V];
#pragma unroll
    for (int v = 0; v < V; v++) a[v] = 0.0f;
    if (c < D) {
      if (sub == 0) load_vec<V>(partial + (2 * (b - 1) + 1) * (int64_t)D + c, a);
      int64_t k = lo;
      for (; k + 7 < hi; k += 8) {
        float p[8][V];
#pragma unroll
        for (int u = 0; u < 8; u++) load_vec<V>(partial + 2 * (k + u) * (int64_t)D + c, p[u]);
#pragma unroll
        for (int v = 0; v < V; v++) a[v] += ((p[0][v] + p[1][v]) + (p[2][v] + p[3][v])) + ((p[4][v] + p[5][v]) + (p[6][v] + p[7][v]));
      }
      for (; k < hi; k++) {
        float p[V];
        load_vec<V>(partial + 2 * k * (int64_t)D + c, p);
#pragma unroll
        for (int v = 0; v < V; v++) a[v] += p[v];
      }
    }
    store_vec<V>(&sum[sub][col * V], a);
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * V; e += kBlock) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; k++) s += sum[k][e];
      if (c0 + e < D) dtable[(int64_t)key * D + c0 + e] = from_f32<T>(s * scale);
    }
    __syncthreads();
  }
}

static int lanes_for(int64_t vecs) {
  int G = 1;
  while (G < vecs && G < kBlock) G <<= 1;
  return G;
}
static int key_bits(int64_t V) {  // keys 0 .. V
  int b = 1;
  while (((int64_t)1 << b) <= V) b++;
  return b;
}
// Positions a chunk: enough chunks for the card, and for very long lists few enough that a frequent token's partial sums stay few.
static int chunk_of(int64_t n) { return n <= (1 << 20) ? 32 : 64; }

struct SortPlan {
  int passes, bits, tile;
  int64_t blocks;
};
static SortPlan sort_plan(int64_t n, int64_t V) {
  SortPlan p;
  const int kb = key_bits(V);
  p.passes = (kb + kSortBits - 1) / kSortBits;
  p.bits = (kb + p.passes - 1) / p.passes;
  int64_t tile = 2 * kSortWaves * kWave;  // 128 positions a wave at least
  while ((n + tile - 1) / tile > kSortBlocks) tile *= 2;
  p.tile = (int)tile;
  p.blocks = (n + tile - 1) / tile;
  return p;
}
struct BwdLayout { size_t key[2], pos[2], hist, partial, total; };
static BwdLayout bwd_layout(int64_t n, int64_t V, int64_t D) {
  BwdLayout L;
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t o = at; at += round_up(bytes, 256); return o; };
  const bool small = n <= kSortSmall;
  for (int i = 0; i < 2; i++) {
    L.key[i] = take(i && small ? 0 : (size_t)n * 4);
    L.pos[i] = take(i && small ? 0 : (size_t)n * 4);
  }
  const SortPlan p = sort_plan(n, V);
  L.hist = take(small ? 0 : (size_t)p.blocks * (1u << p.bits) * 4);
  const int chunk = chunk_of(n);
  L.partial = take((size_t)((n + chunk - 1) / chunk) * 2 * D * 4);
  L.total = at;
  return L;
}

template <typename T, typename I>
static int fwd(int64_t n, int64_t V, int64_t D, const void *ids, const void *table, int64_t ld, float scale, void *out, hipStream_t st) {
  const bool vec = D % kVec<T> == 0 && ld % kVec<T> == 0 && aligned_to(table, 16) && aligned_to(out, 16);
  const int G = lanes_for((D + kVec<T> - 1) / kVec<T>);
  const int64_t blocks = (n + kBlock / G - 1) / (kBlock / G);
  if (!grid_ok(blocks)) return DGS_ERANGE;
  if (vec)
    hipLaunchKernelGGL((embedding_fwd_kernel<T, I, true>), dim3((unsigned)blocks), dim3(kBlock), 0, st, n, V, (int)D, G, (const I *)ids, (const T *)table, ld, scale, (T *)out);
  else
    hipLaunchKernelGGL((embedding_fwd_kernel<T, I, false>), dim3((unsigned)blocks), dim3(kBlock), 0, st, n, V, (int)D, G, (const I *)ids, (const T *)table, ld, scale, (T *)out);
  return check_launch();
}

template <typename I>
static int sort_ids(int64_t n, int64_t V, int64_t pad, const I *ids, char *ws, const BwdLayout &L, uint32_t **key, int **pos, hipStream_t st) {
  if (n <= kSortSmall) {
    *key = (uint32_t *)(ws + L.key[0]);
    *pos = (int *)(ws + L.pos[0]);
    hipLaunchKernelGGL((embedding_rank_kernel<I>), dim3((unsigned)((n + 15) / 16)), dim3(kBlock), 0, st, (int)n, V, pad, ids, *key, *pos);
    return check_launch();
  }
  const SortPlan p = sort_plan(n, V);
  int *hist = (int *)(ws + L.hist);
  const dim3 grid((unsigned)p.blocks), block(kSortWaves * kWave);
  const uint32_t *kin = nullptr;
  const int *pin = nullptr;
  for (int i = 0; i < p.passes; i++) {
    uint32_t *kout = (uint32_t *)(ws + L.key[i & 1]);
    int *pout = (int *)(ws + L.pos[i & 1]);
    hipLaunchKernelGGL((embedding_count_kernel<I>), grid, block, 0, st, n, V, pad, p.tile, i * p.bits, p.bits, ids, kin, hist);
    hipLaunchKernelGGL((embedding_place_kernel<I>), grid, block, 0, st, n, V, pad, p.tile, i * p.bits, p.bits, ids, kin, pin, hist, kout, pout);
    if (check_launch() != DGS_OK) return DGS_ELAUNCH;
    kin = kout;
    pin = pout;
    *key = kout;
    *pos = pout;
  }
  return DGS_OK;
}

template <typename T>
static int bwd(int64_t n, int64_t V, int64_t D, const uint32_t *key, const int *pos, const void *dout, int64_t ldo, float scale, void *dtable, float *partial,
               hipStream_t st) {
  const bool vec = D % kVec<T> == 0 && ldo % kVec<T> == 0 && aligned_to(dout, 16) && aligned_to(dtable, 16);
  const int64_t vecs = (D + kVec<T> - 1) / kVec<T>;
  const int G = lanes_for(vecs) < kLeastLanes ? kLeastLanes : lanes_for(vecs), chunk = chunk_of(n);
  const int64_t n_chunks = (n + chunk - 1) / chunk, per = kBlock / G, tiles = (vecs + G - 1) / G;
  // a clearing workgroup writes about 64 KB; its rows go by a bit map of 256
  const int64_t rowb = D * (int64_t)sizeof(T);
  const int fill_rows = (int)(65536 / rowb < 1 ? 1 : 65536 / rowb > 256 ? 256 : 65536 / rowb);
  const int64_t fill = (V + fill_rows - 1) / fill_rows, work = (n_chunks + per - 1) / per * tiles;
  if (!grid_ok(fill + work)) return DGS_ERANGE;
  // zeros past the caches up to the last level's 256 MB (an 87 MB table: 46 us, through them 52), through them beyond (1 GB: 219 us, past 249)
  const int keep = V * rowb > ((int64_t)256 << 20);
  const dim3 grid((unsigned)(work + fill));
  if (vec)
    hipLaunchKernelGGL((embedding_bwd_kernel<T, true>), grid, dim3(kBlock), 0, st, n, V, (int)D, G, chunk, n_chunks, (int)tiles, work, fill_rows, keep, key, pos, (const T *)dout, ldo, scale, (T *)dtable, partial);
  else
    hipLaunchKernelGGL((embedding_bwd_kernel<T, false>), grid, dim3(kBlock), 0, st, n, V, (int)D, G, chunk, n_chunks, (int)tiles, work, fill_rows, keep, key, pos, (const T *)dout, ldo, scale, (T *)dtable, partial);
  if (check_launch() != DGS_OK) return DGS_ELAUNCH;
  const int64_t cols = (D + 31) / 32, most = 0xffffffffll / kBlock;  // (a launch holds 2^24 - 1 workgroups in a row)
  for (int64_t first = 1; first < n_chunks; first += most) {
    const unsigned borders = (unsigned)(n_chunks - first < most ? n_chunks - first : most);
    if (D % 4 == 0)
      hipLaunchKernelGGL((embedding_join_kernel<T, 4>), dim3(borders, (unsigned)((cols + 3) / 4 < 16 ? (cols + 3) / 4 : 16)), dim3(kBlock), 0, st, first, V, (int)D, chunk, n_chunks, key,
                         scale, partial, (T *)dtable);
    else
      hipLaunchKernelGGL((embedding_join_kernel<T, 1>), dim3(borders, (unsigned)(cols < 16 ? cols : 16)), dim3(kBlock), 0, st, first, V, (int)D, chunk, n_chunks, key, scale, partial,
                         (T *)dtable);
    if (check_launch() != DGS_OK) return DGS_ELAUNCH;
  }
  return DGS_OK;
}

}  // namespace dgs

using namespace dgs;

static int embedding_sizes(int dtype, int id_bytes, int64_t n, int64_t V, int64_t D) {
  if (!dtype_ok(dtype) || (id_bytes != 4 && id_bytes != 8) || n < 0 || V < 0 || D <= 0) return DGS_EINVAL;
  if (n >= INT32_MAX || V >= INT32_MAX || D >= INT32_MAX / 64) return DGS_ERANGE;
  return DGS_OK;
}

extern "C" int dgs_embedding(int dtype, int id_bytes, int64_t n, int64_t V, int64_t D, const void *ids, const void *table, int64_t ld_table, float scale,
                             void *out, dgsStream_t stream) {
  const int rc = embedding_sizes(dtype, id_bytes, n, V, D);
  if (rc != DGS_OK) return rc;
  if (n == 0) return DGS_OK;
  if (!ids || !out || (V > 0 && !table) || ld_table < 0) return DGS_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
#define DGS_GO(T) return id_bytes == 8 ? fwd<T, int64_t>(n, V, D, ids, table, ld_table, scale, out, st) : fwd<T, int32_t>(n, V, D, ids, table, ld_table, scale, out, st)
  if (dtype == DGS_F32) DGS_GO(float);
  if (dtype == DGS_F16) DGS_GO(f16);
  DGS_GO(bf16);
#undef DGS_GO
}

extern "C" size_t dgs_embedding_bwd_workspace_bytes(int64_t n, int64_t V, int64_t D) {
  if (embedding_sizes(DGS_F32, 4, n, V, D) != DGS_OK) return 0;  // (sizes that the entry refuses)
  if (n == 0) return 256;
  return bwd_layout(n, V, D).total;
}

extern "C" int dgs_embedding_bwd(int dtype, int id_bytes, int64_t n, int64_t V, int64_t D, const void *ids, int64_t padding_idx, const void *dout, int64_t ld_dout,
                                 float scale, void *dtable, void *workspace, size_t workspace_bytes, dgsStream_t stream) {
  const int rc = embedding_sizes(dtype, id_bytes, n, V, D);
  if (rc != DGS_OK) return rc;
  if (V == 0) return DGS_OK;
  if (!dtable || (n > 0 && (!ids || !dout || ld_dout < 0))) return DGS_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  uint32_t *key = nullptr;
  int *pos = nullptr;
  float *partial = nullptr;
  if (n > 0) {
    if (!workspace || workspace_bytes < dgs_embedding_bwd_workspace_bytes(n, V, D)) return DGS_EWORKSPACE;
    char *ws = static_cast<char *>(workspace);
    const BwdLayout L = bwd_layout(n, V, D);
    partial = (float *)(ws + L.partial);
    const int r = id_bytes == 8 ? sort_ids<int64_t>(n, V, padding_idx, (const int64_t *)ids, ws, L, &key, &pos, st)
                                : sort_ids<int32_t>(n, V, padding_idx, (const int32_t *)ids, ws, L, &key, &pos, st);
    if (r != DGS_OK) return r;
  }
  if (dtype == DGS_F32) return bwd<float>(n, V, D, key, pos, dout, ld_dout, scale, dtable, partial, st);
  if (dtype == DGS_F16) return bwd<f16>(n, V, D, key, pos, dout, ld_dout, scale, dtable, partial, st);
  return bwd<bf16>(n, V, D, key, pos, dout, ld_dout, scale, dtable, partial, st);
}
