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
// Bound by HBM.  A thread owns 16 consecutive columns: 32 bytes of each 16-bit
// operand and one 16-byte vector of each q; two neighbouring lanes share a
// group.  Every operand is touched once (nontemporal).  Rows need no
// alignment: global memory takes 16-byte accesses at any element's address.
#include "gelu.h"

#include "common.h"

namespace {

constexpr int kBlock = 256;
constexpr int kOwn = 16;    // columns of a thread
constexpr int kGroup = 32;  // columns that share a scale

// 16 bytes at an address that is a multiple of the element only
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <class T>
__device__ __forceinline__ void load_own(const T* p, int n, float (&v)[kOwn]) {
  constexpr int PER = 16 / (int)sizeof(T);
  if (n >= kOwn) {
    Vec16<T> t[kOwn / PER];
#pragma unroll
    for (int k = 0; k < kOwn / PER; ++k) {
      const u32x4_any w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p + k * PER));
      t[k].raw = make_uint4(w.x, w.y, w.z, w.w);
    }
#pragma unroll
    for (int j = 0; j < kOwn; ++j) v[j] = to_f32(t[j / PER].v[j % PER]);
  } else {
#pragma unroll
    for (int j = 0; j < kOwn; ++j) v[j] = j < n ? to_f32(p[j]) : 0.f;
  }
}

template <class T>
__device__ __forceinline__ void store_own(T* p, int n, const float (&v)[kOwn]) {
  constexpr int PER = 16 / (int)sizeof(T);
  if (n >= kOwn) {
#pragma unroll
    for (int k = 0; k < kOwn / PER; ++k) {
      Vec16<T> t;
#pragma unroll
      for (int j = 0; j < PER; ++j) t.v[j] = from_f32<T>(v[k * PER + j]);
      const u32x4_any w = {t.raw.x, t.raw.y, t.raw.z, t.raw.w};
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any*>(p + k * PER));
    }
  } else {
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
      if (j < n) p[j] = from_f32<T>(v[j]);
  }
}

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

// A thread's 16 values in 8 bits: q, and the group's e + 127.
__device__ __forceinline__ uint4 keep(const float (&x)[kOwn], uint32_t& scale) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    const float t = fabsf(x[j]);
    m = fmaxf(m, t < INFINITY ? t : 0.f);  // infinities and NaN do not count
  }
  m = fmaxf(m, __shfl_xor(m, 1, 64));  // the group's other lane
  // m = f 2^(b - 127) with f in [1, 2): 127 * 2^e >= m from e = b - 133 on, or
  // one more where f > 127 / 64
  const uint32_t bits = __float_as_uint(m);
  int e = (int)(bits >> 23) - 133 + ((bits & 0x7fffff) > 0x7e0000 ? 1 : 0);
  e = e < -126 ? -126 : e;
  scale = (uint32_t)(e + 127);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  uint32_t q[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float v = x[4 * k + j];
      // v / 2^e + 1.5 * 2^23 rounds to an integer, to even, in the low bits
      const uint32_t r = __float_as_uint(fmaf(v, inv, 12582912.f));
      const uint32_t b = fabsf(v) < INFINITY ? r & 0xff : 0x80u;
      w |= b << (8 * j);
    }
    q[k] = w;
  }
  return make_uint4(q[0], q[1], q[2], q[3]);
}

__device__ __forceinline__ void kept_values(const uint4& q, uint32_t scale, float (&v)[kOwn]) {
  const float s = __uint_as_float(scale << 23);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    const int b = (int8_t)(w[j / 4] >> (8 * (j % 4)));
    v[j] = b == -128 ? __builtin_nanf("") : (float)b * s;
  }
}

struct Args {
  const void* gate; int64_t ld_gate;
  const void* up; int64_t ld_up;
  void* out; int64_t ld_out;       // backward: the gradient of the output (read)
  void* dgate; void* dup; int64_t ld_grad;
  uint8_t* kept;
  uint32_t n, per_row;             // threads' pieces: in all, and of a row (even)
  uint32_t rows, cols;
};

__device__ __forceinline__ uint8_t* kept_q(const Args& a, uint32_t i, bool up) {
  return a.kept + ((int64_t)(up ? a.n : 0) + i) * kOwn;
}

__device__ __forceinline__ uint16_t* kept_scales(const Args& a, uint32_t i) {
  return reinterpret_cast<uint16_t*>(a.kept + (int64_t)2 * a.n * kOwn) + (i >> 1);
}

template <class T, int ACT, bool KEEP>
__global__ __launch_bounds__(kBlock) void glu_act8_fwd_kernel(Args a) {
  const uint32_t i = blockIdx.x * kBlock + threadIdx.x;
  if (i >= a.n) return;  // (n is even: both lanes of a group)
  const uint32_t r = i / a.per_row, c = (i - r * a.per_row) * kOwn;
  const int left = (int)a.cols - (int)c;  // <= 0 in the second half of a last, short group
  float g[kOwn], u[kOwn], o[kOwn];
  load_own((const T*)a.gate + (int64_t)r * a.ld_gate + c, left, g);
  load_own((const T*)a.up + (int64_t)r * a.ld_up + c, left, u);
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    float act, slope;
    act_and_slope<ACT>(g[j], act, slope);
    o[j] = act * u[j];
  }
  store_own((T*)a.out + (int64_t)r * a.ld_out + c, left, o);
  if constexpr (KEEP) {
    uint32_t sg, su;
    const uint4 qg = keep(g, sg), qu = keep(u, su);
    Vec16<uint8_t> t;
    t.raw = qg;
    store16_nt(kept_q(a, i, false), t);
    t.raw = qu;
    store16_nt(kept_q(a, i, true), t);
    if (!(i & 1)) *kept_scales(a, i) = (uint16_t)(sg | su << 8);
  }
}

template <class T, int ACT>
__global__ __launch_bounds__(kBlock) void glu_act8_bwd_kernel(Args a) {
  const uint32_t i = blockIdx.x * kBlock + threadIdx.x;
  if (i >= a.n) return;
  const uint32_t r = i / a.per_row, c = (i - r * a.per_row) * kOwn;
  const int left = (int)a.cols - (int)c;
  const Vec16<uint8_t> qg = load16_nt(kept_q(a, i, false)), qu = load16_nt(kept_q(a, i, true));
  const uint32_t scales = *kept_scales(a, i);
  float d[kOwn], g[kOwn], u[kOwn];
  load_own((const T*)a.out + (int64_t)r * a.ld_out + c, left, d);
  kept_values(qg.raw, scales & 0xff, g);
  kept_values(qu.raw, scales >> 8, u);
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    float act, slope;
    act_and_slope<ACT>(g[j], act, slope);
    g[j] = d[j] * u[j] * slope;
    u[j] = d[j] * act;
  }
  store_own((T*)a.dgate + (int64_t)r * a.ld_grad + c, left, g);
  store_own((T*)a.dup + (int64_t)r * a.ld_grad + c, left, u);
}

int64_t pieces(int64_t cols) { return (cols + kGroup - 1) / kGroup * (kGroup / kOwn); }

template <class T, int ACT>
int launch(const Args& a, bool bwd, hipStream_t s) {
  const unsigned grid = (a.n + kBlock - 1) / kBlock;
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
  const int64_t lim = 0x40000000;  // pieces of a call, and the threads of its grid, stay below 2^31
  if (rows > lim || cols > lim || rows * pieces(cols) > lim)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: more than 2^34 values in a call", what);
  a.rows = (uint32_t)rows;
  a.cols = (uint32_t)cols;
  a.per_row = (uint32_t)pieces(cols);
  a.n = a.rows * a.per_row;
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
  const int64_t n = rows * pieces(cols);
  return 2 * n * kOwn + n / 2 * 2;
}

extern "C" int forge_glu_act8_fwd(int dtype, int activation, const void* gate, int64_t ld_gate, const void* up,
                                  int64_t ld_up, void* out, int64_t ld_out, void* kept, int64_t rows, int64_t cols,
                                  void* stream) {
  Args a = {};
  if (int rc = prepare("glu_act8_fwd", dtype, activation, rows, cols, a)) return rc;
  if (a.n == 0) return FORGE_OK;
  if (ld_gate < cols || ld_up < cols || ld_out < cols)
    return forge_set_error(FORGE_ERR_INVALID, "glu_act8_fwd: leading dimension smaller than cols");
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
  if (!kept) return forge_set_error(FORGE_ERR_INVALID, "glu_act8_bwd: kept is NULL");
  if (!element_aligned(dout, dtype) || !element_aligned(dgate, dtype) || !element_aligned(dup, dtype) || !aligned16(kept))
    return forge_set_error(FORGE_ERR_INVALID, "glu_act8_bwd: misaligned pointer");
  a.out = const_cast<void*>(dout); a.ld_out = ld_dout;
  a.kept = (uint8_t*)const_cast<void*>(kept);
  a.dgate = dgate; a.dup = dup; a.ld_grad = ld_grad;
  return dispatch(a, dtype, activation, true, stream);
}
