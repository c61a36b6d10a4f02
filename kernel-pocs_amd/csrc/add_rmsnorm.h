// What the kernels of the norm with the residual's addition and of 8-bit rows
// share: a thread's columns of a row, and sums over the threads of a row.
//
// TPR threads (64: a wave, otherwise a workgroup) take a row of H values in vectors of
// V = 16 bytes: thread t the vectors t, t + TPR, ... (NV of them, held in registers;
// NV = 0: any number, read again where they are needed).  Rows may begin at any
// element: global memory takes 16-byte accesses at any address.  The last vector of
// a row may be short.
#pragma once

#include <type_traits>

#include "common.h"

namespace frows {

typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

template <class T> constexpr int V = 16 / (int)sizeof(T);

// V values of a row, held as words (a 16-bit value in a register of its own
// would take all of it)
template <class T>
struct Vec {
  uint32_t w[4];
  __device__ __forceinline__ float get(int i) const {
    if constexpr (std::is_same_v<T, float>) return __uint_as_float(w[i]);
    else if constexpr (std::is_same_v<T, bf16_t>) return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return (float)__builtin_bit_cast(fp16_t, (uint16_t)(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
  }
  __device__ __forceinline__ void set(const float* f) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef T t2 __attribute__((ext_vector_type(2)));
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{f[2 * i], f[2 * i + 1]}), t2));
    }
  }
  // values widened before this point are not kept behind it: they are widened again
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(w[i]));
  }
  __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0; }
};

template <class T> struct Raw { typedef uint16_t type; };
template <> struct Raw<float> { typedef uint32_t type; };

// 16 bytes of a row, of which `n` values exist (the rest are zeros).  A row is
// read once: nontemporal.
template <class T>
__device__ __forceinline__ Vec<T> load_part(const T* p, int n) {
  Vec<T> r;
  if (n >= V<T>) {
    const u32x4_any w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
    r.w[0] = w.x; r.w[1] = w.y; r.w[2] = w.z; r.w[3] = w.w;
  } else {
    typedef typename Raw<T>::type R;
    const R* e = reinterpret_cast<const R*>(p);
    r.clear();
#pragma unroll
    for (int i = 0; i < V<T>; ++i)
      if (i < n) r.w[i * sizeof(R) / 4] |= (uint32_t)e[i] << (sizeof(R) == 2 ? 16 * (i % 2) : 0);
  }
  return r;
}

// Loads of a row that is held, without branches: only then can the compiler wait for
// one row's loads while the next one's are in flight (of loads that may not have been
// made it has to wait for all).  Vectors that do not exist are the last one again,
// rows the last row; a short last vector is read from V values before the row's
// end (rows of less than V values are not held) and moved into place by fit().
template <class T>
__device__ __forceinline__ Vec<T> load_held(const T* row, int c, int64_t H) {
  const u32x4_any w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(row + min((int64_t)c, H - V<T>)));
  Vec<T> r;
  r.w[0] = w.x; r.w[1] = w.y; r.w[2] = w.z; r.w[3] = w.w;
  return r;
}
template <class T>
__device__ __forceinline__ void fit(Vec<T>& r, int n) {
  if (n >= V<T>) return;
  unsigned __int128 x = __builtin_bit_cast(unsigned __int128, r) >> (8 * (int)sizeof(T) * (V<T> - n));
  r = __builtin_bit_cast(Vec<T>, x);
}

template <class T>
__device__ __forceinline__ void store_part(T* p, const Vec<T>& r, int n) {
  if (n >= V<T>) {
    const u32x4_any w = {r.w[0], r.w[1], r.w[2], r.w[3]};
    *reinterpret_cast<u32x4_any*>(p) = w;
  } else {
    typedef typename Raw<T>::type R;
    R* e = reinterpret_cast<R*>(p);
#pragma unroll
    for (int i = 0; i < V<T>; ++i)
      if (i < n) e[i] = (R)(r.w[i * sizeof(R) / 4] >> (sizeof(R) == 2 ? 16 * (i % 2) : 0));
  }
}

// N values of type S at any element, widened
template <class S, int N>
__device__ __forceinline__ void load_wide(const S* p, float* o) {
  constexpr int PER = 16 / (int)sizeof(S);
  if constexpr (N >= PER) {
#pragma unroll
    for (int k = 0; k < N / PER; ++k) {
      Vec16<S> v;
      const u32x4_any w = *reinterpret_cast<const u32x4_any*>(p + k * PER);
      v.raw = make_uint4(w.x, w.y, w.z, w.w);
#pragma unroll
      for (int i = 0; i < PER; ++i) o[k * PER + i] = to_f32(v.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = to_f32(p[i]);
  }
}

// V values of a weight of any type, widened (NULL: ones)
template <class T>
__device__ __forceinline__ void load_weight(const void* w, int w_dtype, int64_t c, int n, float (&o)[V<T>]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < V<T>; ++i) o[i] = 1.f;
  } else if (n >= V<T>) {
    if (w_dtype == FORGE_DTYPE_F32) load_wide<float, V<T>>((const float*)w + c, o);
    else if (w_dtype == FORGE_DTYPE_F16) load_wide<fp16_t, V<T>>((const fp16_t*)w + c, o);
    else load_wide<bf16_t, V<T>>((const bf16_t*)w + c, o);
  } else {
#pragma unroll
    for (int i = 0; i < V<T>; ++i) {
      if (i >= n) o[i] = 0.f;
      else if (w_dtype == FORGE_DTYPE_F32) o[i] = ((const float*)w)[c + i];
      else if (w_dtype == FORGE_DTYPE_F16) o[i] = (float)((const fp16_t*)w)[c + i];
      else o[i] = (float)((const bf16_t*)w)[c + i];
    }
  }
}

// op over the 64 lanes of a wave, in a fixed order: within rows of 16 lanes by
// data-parallel moves, then over the four rows.  (By ds_bpermute, a trip to LDS a
// step, a row of 8 bits waits longest for this.)
template <int CTRL, class A>
__device__ __forceinline__ A moved(A v) {
  if constexpr (sizeof(A) == 8) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = moved<CTRL>((uint32_t)x), hi = moved<CTRL>((uint32_t)(x >> 32));
    return __builtin_bit_cast(A, (uint64_t)hi << 32 | lo);
  } else {
    return __builtin_bit_cast(A, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
  }
}
template <class A>
__device__ __forceinline__ A lane_value(A v, int lane) {
  if constexpr (sizeof(A) == 8) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = lane_value((uint32_t)x, lane), hi = lane_value((uint32_t)(x >> 32), lane);
    return __builtin_bit_cast(A, (uint64_t)hi << 32 | lo);
  } else {
    return __builtin_bit_cast(A, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  }
}
template <class A, class Op>
__device__ __forceinline__ A over_wave(A v, Op op) {
  v = op(v, moved<0xb1>(v));   // lane ^ 1
  v = op(v, moved<0x4e>(v));   // lane ^ 2
  v = op(v, moved<0x141>(v));  // the other half of 8
  v = op(v, moved<0x140>(v));  // the other half of 16
  return op(op(lane_value(v, 0), lane_value(v, 16)), op(lane_value(v, 32), lane_value(v, 48)));
}

// Sum over the TPR threads of a row, in a fixed order; every thread gets it.
// buf: one slot per wave, used by one call between two barriers.
template <int TPR, class A>
__device__ __forceinline__ A row_sum(A v, A* buf) {
  v = over_wave(v, [](A a, A b) { return a + b; });
  if constexpr (TPR == 64) return v;
  if (threadIdx.x % 64 == 0) buf[threadIdx.x / 64] = v;
  __syncthreads();
  v = buf[0];
#pragma unroll
  for (int w = 1; w < TPR / 64; ++w) v += buf[w];
  return v;
}

template <int TPR> constexpr int threads_of = TPR > 256 ? TPR : 256;
template <int TPR> constexpr int rows_per_block = threads_of<TPR> / TPR;

// The kernel F<T, TPR, NV, ...> for rows of H values, and its threads.
#define FROWS_PICK(T, H, F, ...)                                \
  do {                                                          \
    const int64_t nv_ = ((H) + frows::V<T> - 1) / frows::V<T>;  \
    if ((H) < frows::V<T>) return F<T, 256, 0, __VA_ARGS__>;    \
    if (nv_ <= 64) return F<T, 64, 1, __VA_ARGS__>;             \
    if (nv_ <= 128) return F<T, 64, 2, __VA_ARGS__>;            \
    if (nv_ <= 256) return F<T, 256, 1, __VA_ARGS__>;           \
    if (nv_ <= 512) return F<T, 256, 2, __VA_ARGS__>;           \
    if (nv_ <= 1024) return F<T, 512, 2, __VA_ARGS__>;          \
    if (nv_ <= 2048) return F<T, 1024, 2, __VA_ARGS__>;         \
    return F<T, 256, 0, __VA_ARGS__>;                           \
  } while (0)

// (host) rows that a workgroup of that kernel takes at once, and its threads
inline int rows_at_once(int64_t H, int size) { return H >= 16 / size && H * size <= 128 * 16 ? 4 : 1; }
inline int threads_for(int64_t H, int size) {
  const int64_t nv = (H * size + 15) / 16;
  return nv <= 512 || nv > 2048 ? 256 : nv <= 1024 ? 512 : 1024;
}

}  // namespace frows
