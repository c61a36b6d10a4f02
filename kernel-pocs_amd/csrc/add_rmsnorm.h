// What the kernels of the norm with the residual's addition and of 8-bit rows
// share: a thread's columns of a row, and sums over the threads of a row.
//
// TPR threads (64: a wave, 256: a workgroup) take a row of H values in vectors of
// V = 16 bytes: thread t the vectors t, t + TPR, ... (NV of them, held in registers;
// NV = 0: any number, read again where they are needed).  Rows may begin at any
// element: global memory takes 16-byte accesses at any address, and they
// measured as fast as aligned ones.  The last vector of a row may be short.
#pragma once

#include <type_traits>

#include "common.h"

namespace frows {

typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

template <class T> constexpr int V = 16 / (int)sizeof(T);

// 16 bytes of a row, of which `n` values exist (the rest are zeros)
template <class T>
__device__ __forceinline__ Vec16<T> load_part(const T* p, int n) {
  Vec16<T> r;
  if (n >= V<T>) {
    const u32x4_any w = *reinterpret_cast<const u32x4_any*>(p);
    r.raw = make_uint4(w.x, w.y, w.z, w.w);
  } else {
    r.raw = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < V<T>; ++i)
      if (i < n) r.v[i] = p[i];
  }
  return r;
}

template <class T>
__device__ __forceinline__ void store_part(T* p, const Vec16<T>& r, int n) {
  if (n >= V<T>) {
    const u32x4_any w = {r.raw.x, r.raw.y, r.raw.z, r.raw.w};
    *reinterpret_cast<u32x4_any*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < V<T>; ++i)
      if (i < n) p[i] = r.v[i];
  }
}

// V values of a weight of any type, widened
template <class T>
__device__ __forceinline__ void load_weight(const void* w, int w_dtype, int64_t c, int n, float (&o)[V<T>]) {
#pragma unroll
  for (int i = 0; i < V<T>; ++i) {
    if (i >= n) o[i] = 0.f;
    else if (!w) o[i] = 1.f;
    else if (w_dtype == FORGE_DTYPE_F32) o[i] = ((const float*)w)[c + i];
    else if (w_dtype == FORGE_DTYPE_F16) o[i] = (float)((const fp16_t*)w)[c + i];
    else o[i] = (float)((const bf16_t*)w)[c + i];
  }
}

// Sum over the TPR threads of a row, in a fixed order; every thread gets it.
// buf: one slot per wave, used by one call between two barriers.
template <int TPR, class A>
__device__ __forceinline__ A row_sum(A v, A* buf) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (TPR == 64) return v;
  if (threadIdx.x % 64 == 0) buf[threadIdx.x / 64] = v;
  __syncthreads();
  v = buf[0];
#pragma unroll
  for (int w = 1; w < TPR / 64; ++w) v += buf[w];
  return v;
}

template <int TPR>
constexpr int rows_per_block = 256 / TPR;

// Launches f<TPR, NV> for rows of H values.
#define FROWS_PICK(T, H, F)                                     \
  do {                                                          \
    const int64_t nv_ = ((H) + frows::V<T> - 1) / frows::V<T>;  \
    if (nv_ <= 64) return F<T, 64, 1>;                          \
    if (nv_ <= 128) return F<T, 64, 2>;                         \
    if (nv_ <= 256) return F<T, 256, 1>;                        \
    if (nv_ <= 512) return F<T, 256, 2>;                        \
    if (nv_ <= 1024) return F<T, 256, 4>;                       \
    if (nv_ <= 2048) return F<T, 256, 8>;                       \
    return F<T, 256, 0>;                                        \
  } while (0)

}  // namespace frows
