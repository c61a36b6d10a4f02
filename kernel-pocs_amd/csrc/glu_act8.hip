// Gated activation out = act(gate) * up that keeps gate and up in 8 bits for
// its backward pass, for gfx950.
//
// What is kept: groups of 32 consecutive values of a row share a power of two
// 2^e, the least one with |x| <= 127 * 2^e in the group (e >= -126), and each
// value is the integer q = round(x / 2^e) to even, |q| <= 127.  x / 2^e and
// q * 2^e are exact in fp32, so what is kept depends on x alone, and its error
// is at most half of 2^e: 1/127 to 1/254 of the group's largest value.  An
// infinity or NaN is kept as q = -128, which comes back as NaN, and does not
// count for e.  With g, u the kept values the backward is
//     dgate = dout u act'(g),   dup = dout act(g),
// and the forward uses gate and up as they came.  8.5 bits a value instead of
// 16 or 32 stay between the passes; the traffic of a step is the same.
//
// Buffer of a call ("kept"): q of gate [rows][pitch], q of up [rows][pitch]
// with pitch = cols rounded up to 32, then [rows][pitch / 32] pairs of bytes
// e + 127 (gate's, up's).
//
// Bound by HBM.  A thread owns one 16-byte vector of each operand (8 columns, 4
// of fp32), so that a wave's accesses are whole lines, and 8 (4) bytes of each
// q; 4 (8) neighbouring lanes share a group.  Every operand is touched once
// (nontemporal).  Rows need no alignment: global memory takes 16-byte accesses
// at any element's address.  Measured on MI355X, nothing cached, forward /
// backward: bf16 [8192, 14336] silu 161 / 157 us (5.9 / 6.0 TB/s; a copy 5.8),
// tanh 167 / 165; fp16 [4096, 14337] erf 85 / 89; fp32 [4096, 11008] silu 99 /
// 99.  With 16 columns a thread the 16-bit backward took 237 us (two stores 32
// bytes apart in place of whole lines); one vector in flight 166 / 158, four
// 165 / 159; two in fp32 103 / 107.  The forward's arithmetic (two activations'
// worth) is close behind the memory: testing every value for infinities took
// it to 176 us, so a wave tests its largest and looks closer only then.
#include "gelu.h"

#include "common.h"

namespace {

constexpr int kBlock = 256;
constexpr int kGroup = 32;  // columns that share a scale

// 16 bytes at an address that is a multiple of the element only
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <class T>
struct Own {
  static constexpr int N = 16 / (int)sizeof(T);  // columns of a thread
  static constexpr int LANES = kGroup / N;       // threads of a group
  static constexpr int VECTORS = sizeof(T) == 4 ? 1 : 2;  // in flight for each operand

  static __device__ __forceinline__ Vec16<T> load(const T* p, int n) {
    Vec16<T> t;
    if (n >= N) {
      const u32x4_any w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
      t.raw = make_uint4(w.x, w.y, w.z, w.w);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) t.v[j] = j < n ? p[j] : from_f32<T>(0.f);
    }
    return t;
  }

  static __device__ __forceinline__ void store(T* p, int n, const float (&v)[N]) {
    Vec16<T> t;
#pragma unroll
    for (int j = 0; j < N; ++j) t.v[j] = from_f32<T>(v[j]);
    if (n >= N) {
      const u32x4_any w = {t.raw.x, t.raw.y, t.raw.z, t.raw.w};
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any*>(p));
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n) p[j] = t.v[j];
    }
  }
};

// act(x) and act'(x) in fp32.
template <int ACT>
__device__ __forceinline__ void act_and_slope(float x, float& act, float& slope) {
  if constexpr (ACT == FORGE_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
    act = x * s;
    slope = s * (1.f + x * (1.f - s));
  } else if constexpr (ACT == FORGE_ACT_GELU_TANH) {
    // past 100 the cubic would overflow: tanh is +-1 there
    const bool far = fabsf(x) > 100.f;  // (false for NaN)
    const float xc = far ? copysignf(100.f, x) : x;
    fgelu::gelu_and_grad<true>(xc, act, slope);
    if (far) act = fmaxf(x, 0.f);
  } else {
    fgelu::gelu_and_grad<false>(x, act, slope);
  }
}

template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  const uint32_t w = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
  return v > w ? v : w;
}

// The largest over the lanes of a group of N values a lane: neighbours
// (quad_perm [1, 0, 3, 2]), pairs (quad_perm [2, 3, 0, 1]), and where 8 lanes
// share one the other quad (row_half_mirror).
template <int N>
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
  m = max_dpp<0xb1>(m);
  m = max_dpp<0x4e>(m);
  if constexpr (N == 4) m = max_dpp<0x141>(m);
  return m;
}

constexpr uint32_t kInf = 0x7f800000;

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(b, a, 0x0c0c0400) | __builtin_amdgcn_perm(d, c, 0x04000c0c);
}

// A thread's values in 8 bits: q, and the group's e + 127.  Magnitudes are
// compared as bits, whose order they share, so that one look at the largest
// tells whether a wave has infinities or NaN to leave out.
template <int N>
__device__ __forceinline__ void keep(const float (&x)[N], uint32_t (&q)[N / 4], uint32_t& scale) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t t = __float_as_uint(x[j]) & 0x7fffffff;
    m = m > t ? m : t;
  }
  const bool special = __any(m >= kInf);
  if (special) {
    m = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint32_t t = __float_as_uint(x[j]) & 0x7fffffff;
      m = t < kInf && t > m ? t : m;
    }
  }
  m = group_max<N>(m);
  // m = f 2^(b - 127) with f in [1, 2): 127 * 2^e >= m from e = b - 133 on, or
  // one more where f > 127 / 64
  int e = (int)(m >> 23) - 133 + ((m & 0x7fffff) > 0x7e0000 ? 1 : 0);
  e = e < -126 ? -126 : e;
  scale = (uint32_t)(e + 127);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  uint32_t r[N];
#pragma unroll
  for (int j = 0; j < N; ++j) r[j] = __float_as_uint(fmaf(x[j], inv, 12582912.f));  // rounded to even in the low bits of 1.5 * 2^23 + .
  if (special) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if ((__float_as_uint(x[j]) & 0x7fffffff) >= kInf) r[j] = 0x80;
  }
#pragma unroll
  for (int k = 0; k < N / 4; ++k) q[k] = low_bytes(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
}

template <int N>
__device__ __forceinline__ void kept_values(const uint32_t (&q)[N / 4], uint32_t scale, float (&v)[N]) {
  const float s = __uint_as_float(scale << 23);
  uint32_t hit = 0;  // a byte 0x80 leaves its top bit here (and may leave others')
#pragma unroll
  for (int k = 0; k < N / 4; ++k) {
    const uint32_t t = q[k] ^ 0x80808080u;
    hit |= (t - 0x01010101u) & ~t & 0x80808080u;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = (float)(int8_t)(q[j / 4] >> (8 * (j % 4))) * s;
  if (__any(hit)) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (((q[j / 4] >> (8 * (j % 4))) & 0xff) == 0x80) v[j] = __builtin_nanf("");
  }
}

// q of a thread's columns: N bytes.
template <int N>
__device__ __forceinline__ void load_q(const uint8_t* p, uint32_t (&q)[N / 4]) {
  if constexpr (N == 8) {
    const uint64_t w = __builtin_nontemporal_load(reinterpret_cast<const uint64_t*>(p));
    q[0] = (uint32_t)w;
    q[1] = (uint32_t)(w >> 32);
  } else {
    q[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  }
}

template <int N>
__device__ __forceinline__ void store_q(uint8_t* p, const uint32_t (&q)[N / 4]) {
  if constexpr (N == 8)
    __builtin_nontemporal_store((uint64_t)q[0] | (uint64_t)q[1] << 32, reinterpret_cast<uint64_t*>(p));
  else
    __builtin_nontemporal_store(q[0], reinterpret_cast<uint32_t*>(p));
}

struct Args {
  const void* gate; int64_t ld_gate;
  const void* up; int64_t ld_up;
  void* out; int64_t ld_out;       // backward: the gradient of the output (read)
  void* dgate; void* dup; int64_t ld_grad;
  uint8_t* kept;
  uint32_t n, per_row;             // threads' vectors: in all, and of a row (whole groups)
  uint32_t cols;
};

template <class T>
__device__ __forceinline__ uint8_t* kept_q(const Args& a, uint32_t i, bool up) {
  return a.kept + ((int64_t)(up ? a.n : 0) + i) * Own<T>::N;
}

template <class T>
__device__ __forceinline__ uint16_t* kept_scales(const Args& a, uint32_t i) {
  return reinterpret_cast<uint16_t*>(a.kept + (int64_t)2 * a.n * Own<T>::N) + i / Own<T>::LANES;
}

template <class T, int ACT, bool KEEP>
__global__ __launch_bounds__(kBlock) void glu_act8_fwd_kernel(Args a) {
  using O = Own<T>;
  constexpr int N = O::N, U = O::VECTORS;
  const uint32_t i0 = blockIdx.x * (kBlock * U) + threadIdx.x;
  Vec16<T> g[U], u[U];
  uint32_t row[U];
  int col[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t i = i0 + k * kBlock;
    if (i >= a.n) continue;  // (n is whole groups)
    row[k] = i / a.per_row;
    col[k] = (int)(i - row[k] * a.per_row) * N;
    const int left = (int)a.cols - col[k];  // <= 0 past the end of a last, short group
    g[k] = O::load((const T*)a.gate + (int64_t)row[k] * a.ld_gate + col[k], left);
    u[k] = O::load((const T*)a.up + (int64_t)row[k] * a.ld_up + col[k], left);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t i = i0 + k * kBlock;
    if (i >= a.n) continue;
    float x[N], y[N], o[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      x[j] = to_f32(g[k].v[j]);
      y[j] = to_f32(u[k].v[j]);
      float act, slope;
      act_and_slope<ACT>(x[j], act, slope);
      o[j] = act * y[j];
    }
    O::store((T*)a.out + (int64_t)row[k] * a.ld_out + col[k], (int)a.cols - col[k], o);
    if constexpr (KEEP) {
      uint32_t qx[N / 4], qy[N / 4], sx, sy;
      keep(x, qx, sx);
      keep(y, qy, sy);
      store_q<N>(kept_q<T>(a, i, false), qx);
      store_q<N>(kept_q<T>(a, i, true), qy);
      if (i % O::LANES == 0) *kept_scales<T>(a, i) = (uint16_t)(sx | sy << 8);
    }
  }
}

template <class T, int ACT>
__global__ __launch_bounds__(kBlock) void glu_act8_bwd_kernel(Args a) {
  using O = Own<T>;
  constexpr int N = O::N, U = O::VECTORS;
  const uint32_t i0 = blockIdx.x * (kBlock * U) + threadIdx.x;
  Vec16<T> d[U];
  uint32_t qg[U][N / 4], qu[U][N / 4], scales[U], row[U];
  int col[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t i = i0 + k * kBlock;
    if (i >= a.n) continue;
    row[k] = i / a.per_row;
    col[k] = (int)(i - row[k] * a.per_row) * N;
    d[k] = O::load((const T*)a.out + (int64_t)row[k] * a.ld_out + col[k], (int)a.cols - col[k]);
    load_q<N>(kept_q<T>(a, i, false), qg[k]);
    load_q<N>(kept_q<T>(a, i, true), qu[k]);
    scales[k] = *kept_scales<T>(a, i);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t i = i0 + k * kBlock;
    if (i >= a.n) continue;
    const int left = (int)a.cols - col[k];
    float g[N], u[N];
    kept_values(qg[k], scales[k] & 0xff, g);
    kept_values(qu[k], scales[k] >> 8, u);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float dout = to_f32(d[k].v[j]);
      float act, slope;
      act_and_slope<ACT>(g[j], act, slope);
      g[j] = dout * u[j] * slope;
      u[j] = dout * act;
    }
    O::store((T*)a.dgate + (int64_t)row[k] * a.ld_grad + col[k], left, g);
    O::store((T*)a.dup + (int64_t)row[k] * a.ld_grad + col[k], left, u);
  }
}

int64_t groups_of(int64_t cols) { return (cols + kGroup - 1) / kGroup; }

template <class T, int ACT>
int launch(const Args& a, bool bwd, hipStream_t s) {
  const unsigned per = kBlock * Own<T>::VECTORS, grid = (a.n + per - 1) / per;
  if (bwd) glu_act8_bwd_kernel<T, ACT><<<grid, kBlock, 0, s>>>(a);
  else if (a.kept) glu_act8_fwd_kernel<T, ACT, true><<<grid, kBlock, 0, s>>>(a);
  else glu_act8_fwd_kernel<T, ACT, false><<<grid, kBlock, 0, s>>>(a);
  FORGE_CHECK_LAUNCH();
  return FORGE_OK;
}

template <class T>
int launch_act(const Args& a, int act, bool bwd, hipStream_t s) {
  if (act == FORGE_ACT_SILU) return launch<T, FORGE_ACT_SILU>(a, bwd, s);
  if (act == FORGE_ACT_GELU_TANH) return launch<T, FORGE_ACT_GELU_TANH>(a, bwd, s);
  return launch<T, FORGE_ACT_GELU_ERF>(a, bwd, s);
}

// Sizes shared by both directions; FORGE_OK with a.n == 0 means nothing to do.
int prepare(const char* what, int dtype, int act, int64_t rows, int64_t cols, Args& a) {
  if (rows < 0 || cols < 0) return forge_set_error(FORGE_ERR_INVALID, "%s: negative shape", what);
  if (act != FORGE_ACT_SILU && act != FORGE_ACT_GELU_TANH && act != FORGE_ACT_GELU_ERF)
    return forge_set_error(FORGE_ERR_INVALID, "%s: activation %d", what, act);
  if (dtype != FORGE_DTYPE_F32 && dtype != FORGE_DTYPE_BF16 && dtype != FORGE_DTYPE_F16)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  const int64_t lim = 0x40000000;  // vectors of a call, and the threads of its grid, stay below 2^31
  const int64_t per_row = groups_of(cols) * kGroup * (int64_t)dtype_size(dtype) / 16;
  if (rows > lim || cols > lim || rows * per_row > lim)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: more than 2^30 vectors of 16 bytes in a call", what);
  a.cols = (uint32_t)cols;
  a.per_row = (uint32_t)per_row;
  a.n = (uint32_t)(rows * per_row);
  return FORGE_OK;
}

int dispatch(const Args& a, int dtype, int act, bool bwd, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  if (dtype == FORGE_DTYPE_F32) return launch_act<float>(a, act, bwd, s);
  if (dtype == FORGE_DTYPE_BF16) return launch_act<bf16_t>(a, act, bwd, s);
  return launch_act<fp16_t>(a, act, bwd, s);
}

bool element_aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % dtype_size(dtype) == 0; }

}  // namespace

extern "C" int64_t forge_glu_act8_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  const int64_t n = rows * groups_of(cols);
  return n * (2 * kGroup + 2);
}

extern "C" int forge_glu_act8_fwd(int dtype, int activation, const void* gate, int64_t ld_gate, const void* up,
                                  int64_t ld_up, void* out, int64_t ld_out, void* kept, int64_t rows, int64_t cols,
                                  void* stream) {
  Args a = {};
  if (int rc = prepare("glu_act8_fwd", dtype, activation, rows, cols, a)) return rc;
  if (a.n == 0) return FORGE_OK;
  if (ld_gate < cols || ld_up < cols || ld_out < cols)
    return forge_set_error(FORGE_ERR_INVALID, "glu_act8_fwd: leading dimension smaller than cols");
  if (!gate || !up || !out) return forge_set_error(FORGE_ERR_INVALID, "glu_act8_fwd: a required pointer is NULL");
  if (!element_aligned(gate, dtype) || !element_aligned(up, dtype) || !element_aligned(out, dtype) || !aligned16(kept))
    return forge_set_error(FORGE_ERR_INVALID, "glu_act8_fwd: misaligned pointer");
  a.gate = gate; a.ld_gate = ld_gate;
  a.up = up; a.ld_up = ld_up;
  a.out = out; a.ld_out = ld_out;
  a.kept = (uint8_t*)kept;
  return dispatch(a, dtype, activation, false, stream);
}

extern "C" int forge_glu_act8_bwd(int dtype, int activation, const void* dout, int64_t ld_dout, const void* kept,
                                  void* dgate, void* dup, int64_t ld_grad, int64_t rows, int64_t cols, void* stream) {
  Args a = {};
  if (int rc = prepare("glu_act8_bwd", dtype, activation, rows, cols, a)) return rc;
  if (a.n == 0) return FORGE_OK;
  if (ld_dout < cols || ld_grad < cols)
    return forge_set_error(FORGE_ERR_INVALID, "glu_act8_bwd: leading dimension smaller than cols");
  if (!kept || !dout || !dgate || !dup)
    return forge_set_error(FORGE_ERR_INVALID, "glu_act8_bwd: kept or another required pointer is NULL");
  if (!element_aligned(dout, dtype) || !element_aligned(dgate, dtype) || !element_aligned(dup, dtype) || !aligned16(kept))
    return forge_set_error(FORGE_ERR_INVALID, "glu_act8_bwd: misaligned pointer");
  a.out = const_cast<void*>(dout); a.ld_out = ld_dout;
  a.kept = (uint8_t*)const_cast<void*>(kept);
  a.dgate = dgate; a.dup = dup; a.ld_grad = ld_grad;
  return dispatch(a, dtype, activation, true, stream);
}
