// dense_common.h -- element types, row access and reductions shared by the dense operators (embedding, rms_norm, gated_ffn, fp8).
#pragma once
#include "dgs_common.h"

namespace dgs {

using bf16 = __bf16;
using f16 = _Float16;

// 16 bytes of one row: what a lane moves in one access
template <typename T> constexpr int kVec = 16 / (int)sizeof(T);

typedef uint32_t dgs_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t dgs_u2 __attribute__((ext_vector_type(2)));

template <typename T> __device__ __forceinline__ float to_f32(T x) { return (float)x; }
// one rounding to nearest even, for a value that leaves the kernel in T
template <typename T> __device__ __forceinline__ T from_f32(float x) { return (T)x; }

// kVec elements at p (elements [c, c + kVec) of a row of D): one 16-byte access where the row allows it (VECTOR: pointer, row stride and
// D are multiples of 16 bytes), else element by element with the row's end watched; elements behind it read as 0.
template <typename T, bool VECTOR>
__device__ __forceinline__ void load_row(const T *p, int c, int D, float (&o)[kVec<T>]) {
  constexpr int V = kVec<T>;
  if constexpr (VECTOR) {
    union { dgs_u4 u; T t[V]; } x;
    x.u = *reinterpret_cast<const dgs_u4 *>(p + c);
#pragma unroll
    for (int v = 0; v < V; v++) o[v] = to_f32(x.t[v]);
  } else {
#pragma unroll
    for (int v = 0; v < V; v++) o[v] = c + v < D ? to_f32(p[c + v]) : 0.0f;
  }
}
template <typename T, bool VECTOR>
__device__ __forceinline__ void store_row(T *p, int c, int D, const float (&o)[kVec<T>]) {
  constexpr int V = kVec<T>;
  if constexpr (VECTOR) {
    union { dgs_u4 u; T t[V]; } x;
#pragma unroll
    for (int v = 0; v < V; v++) x.t[v] = from_f32<T>(o[v]);
    *reinterpret_cast<dgs_u4 *>(p + c) = x.u;
  } else {
#pragma unroll
    for (int v = 0; v < V; v++)
      if (c + v < D) p[c + v] = from_f32<T>(o[v]);
  }
}
// the same past the caches: non-temporal
template <typename T, bool VECTOR>
__device__ __forceinline__ void store_row_stream(T *p, int c, int D, const float (&o)[kVec<T>]) {
  constexpr int V = kVec<T>;
  if constexpr (VECTOR) {
    union { dgs_u4 u; T t[V]; } x;
#pragma unroll
    for (int v = 0; v < V; v++) x.t[v] = from_f32<T>(o[v]);
    __builtin_nontemporal_store(x.u, reinterpret_cast<dgs_u4 *>(p + c));
  } else {
    store_row<T, VECTOR>(p, c, D, o);
  }
}

// Sum over the G lanes of a group (G <= 64: lanes of one wave; G = 256: the workgroup, through `red`, 4 floats of LDS per value).
// Every lane gets the same sum, from the same tree.
template <int G>
__device__ __forceinline__ float group_sum(float x, float *red) {
#pragma unroll
  for (int d = 1; d < (G < 64 ? G : 64); d <<= 1) x += __shfl_xor(x, d, 64);
  if constexpr (G > 64) {
    static_assert(G == 256, "a group is a part of a wave or the workgroup");
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return x;
}

// a launch's threads in one dimension are counted in 32 bits
inline bool grid_ok(int64_t blocks, int64_t threads = kBlock) { return blocks * threads <= 0xffffffffll; }
inline bool aligned_to(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline size_t dtype_bytes(int dtype) { return dtype == DGS_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == DGS_F32 || dtype == DGS_F16 || dtype == DGS_BF16; }
inline size_t round_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

}  // namespace dgs
