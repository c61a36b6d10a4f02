// RMS norm with the residual's addition, and rows in 8 bits with one scale each.
//
//   h = round(x + residual)                       (stored: the residual stream)
//   y = round(h rstd (w + offset)),  rstd = 1 / sqrt(mean h^2 + eps)
//   or, in 8 bits, with t = h (w + offset) and a = max |t| of the row:
//   q = round_half_even(127 t / a),  scale = a rstd / 127:  y = q scale
// The integers do not depend on rstd, and both sums of a row are taken in one
// pass.  Rows as they are (no norm): t = x, or x times a scale a column.
//
// The integers are those of exact arithmetic.  t of two 16-bit factors is exact in
// fp32; otherwise the largest is found in 64 bits.  127 t / a errs by less than
// 1e-4 in fp32 (127 times a few roundings of 2^-24), so only values that close
// to a border between two integers are divided again, in 64 bits.
//
// Bound by HBM: x and the residual are read once, h and y written once.
#include "add_rmsnorm.h"

namespace frows {

struct FwdArgs {
  const void* x; int64_t ldx;
  const void* res; int64_t ldr;  // or NULL
  const void* w; int w_dtype;    // or NULL: ones
  void* h;                       // [rows][H], or NULL where there is no residual
  void* y;                       // [rows][H]
  int8_t* q; int64_t ldq;        // [rows][ldq], zeros from H on
  float* scale;                  // [rows]
  float* rstd;                   // [rows], or NULL
  int64_t rows, H;
  float eps, offset;
  int exact;                     // t is exact in fp32
};

enum Mode { NORM, NORM8, ROWS8 };

template <class T, int MODE>
struct Elem {
  // the stored sum
  static __device__ __forceinline__ Vec16<T> add(const Vec16<T>& x, const Vec16<T>& r) {
    Vec16<T> h;
#pragma unroll
    for (int i = 0; i < V<T>; ++i) h.v[i] = from_f32<T>(to_f32(x.v[i]) + to_f32(r.v[i]));
    return h;
  }
};

__device__ __forceinline__ int quantize(float v, float w, float offset, float inv, double a, bool tiny) {
  const float t = v * (w + offset) * inv;
  const float k = rintf(t);
  if (tiny || fabsf(fabsf(t - k) - 0.5f) < 1e-3f) return (int)rint(127.0 * ((double)v * ((double)w + (double)offset)) / a);
  return (int)k;
}

template <class T, int TPR, int NV, int MODE>
__global__ __launch_bounds__(256) void add_rmsnorm_kernel(FwdArgs a) {
  constexpr int VN = V<T>, RPB = rows_per_block<TPR>, N = NV ? NV : 1;
  __shared__ float sums[2][4];
  __shared__ uint32_t tops[2][4];
  __shared__ double tops64[2][4];
  const int tid = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int n_vec = (int)((a.H + VN - 1) / VN);
  const T* xp = (const T*)a.x;
  const T* rp = (const T*)a.res;
  float w[N][VN];
  if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (tid + j * TPR) * VN;
      load_weight<T>(a.w, a.w_dtype, c, (int)(a.H - c), w[j]);
    }
  }
  int flip = 0;
  // (every thread of a workgroup goes through the same rounds: row_sum has barriers)
  for (int64_t first = (int64_t)blockIdx.x * RPB; first < a.rows; first += (int64_t)gridDim.x * RPB, flip ^= 1) {
    const int64_t row = first + slot;
    if (TPR == 64 && row >= a.rows) return;
    Vec16<T> h[N];
    float ss = 0.f;
    uint32_t top = 0;
    double top64 = 0.0;
    auto see = [&](const Vec16<T>& v, const float (&wv)[VN]) {
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        const float f = to_f32(v.v[i]);
        if (MODE != ROWS8) ss += f * f;
        if (MODE != NORM) {
          top = max(top, __float_as_uint(f * (wv[i] + a.offset)) & 0x7fffffffu);
          if (!a.exact) top64 = fmax(top64, fabs((double)f * ((double)wv[i] + (double)a.offset)));
        }
      }
    };
    auto read = [&](int vec) {
      const int c = vec * VN, n = (int)min((int64_t)VN, a.H - c);
      Vec16<T> v = load_part(xp + row * a.ldx + c, n);
      if (MODE != ROWS8 && rp) {
        v = Elem<T, MODE>::add(v, load_part(rp + row * a.ldr + c, n));
        store_part((T*)a.h + row * a.H + c, v, n);
      }
      return v;
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int vec = tid + j * TPR;
        if (vec < n_vec) {
          h[j] = read(vec);
          see(h[j], w[j]);
        }
      }
    } else {
      for (int vec = tid; vec < n_vec; vec += TPR) {
        load_weight<T>(a.w, a.w_dtype, vec * VN, (int)(a.H - vec * VN), w[0]);
        see(read(vec), w[0]);
      }
    }
    float rstd = 1.f;
    if constexpr (MODE != NORM) {
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
      if (!a.exact) {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) top64 = fmax(top64, __shfl_xor(top64, off, 64));
      }
      if constexpr (TPR > 64) {
        if (threadIdx.x % 64 == 0) {
          tops[flip][threadIdx.x / 64] = top;
          tops64[flip][threadIdx.x / 64] = top64;
        }
        if (MODE == ROWS8) __syncthreads();
      }
    }
    if constexpr (MODE != ROWS8) {
      ss = row_sum<TPR>(ss, sums[flip]);
      rstd = rsqrtf(ss / (float)a.H + a.eps);
      if (tid == 0 && a.rstd) a.rstd[row] = rstd;
    }
    float inv = 0.f;
    bool tiny = false, bad = false;
    if constexpr (MODE != NORM) {
      if constexpr (TPR > 64) {
#pragma unroll
        for (int k = 0; k < TPR / 64; ++k) {
          top = max(top, tops[flip][k]);
          top64 = fmax(top64, tops64[flip][k]);
        }
      }
      if (a.exact) top64 = (double)__uint_as_float(top);
      // infinities and NaN: the row's scale is NaN, and so is all that is computed of it
      bad = top >= 0x7f800000u;
      tiny = top64 < 1e-30;
      inv = tiny || bad ? 0.f : 127.f / (float)top64;
      if (tid == 0) a.scale[row] = bad ? __builtin_nanf("") : (float)top64 * rstd / 127.f;
    }
    auto write = [&](const Vec16<T>& v, const float (&wv)[VN], int vec) {
      const int c = vec * VN, n = (int)min((int64_t)VN, a.H - c);
      if constexpr (MODE == NORM) {
        Vec16<T> y;
#pragma unroll
        for (int i = 0; i < VN; ++i) y.v[i] = from_f32<T>(to_f32(v.v[i]) * rstd * (wv[i] + a.offset));
        store_part((T*)a.y + row * a.H + c, y, n);
      } else {
        uint32_t word[VN / 4];
#pragma unroll
        for (int i = 0; i < VN; ++i) {
          const int k = bad || top64 == 0.0 || i >= n ? 0 : quantize(to_f32(v.v[i]), wv[i], a.offset, inv, top64, tiny);
          const uint32_t byte = (uint32_t)(k & 255) << (8 * (i % 4));
          word[i / 4] = i % 4 ? word[i / 4] | byte : byte;
        }
        int8_t* p = a.q + row * a.ldq + c;  // (ldq is a multiple of 16)
        if constexpr (VN == 8) *reinterpret_cast<uint2*>(p) = make_uint2(word[0], word[1]);
        else *reinterpret_cast<uint32_t*>(p) = word[0];
      }
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int vec = tid + j * TPR;
        if (vec < n_vec) write(h[j], w[j], vec);
      }
    } else {
      for (int vec = tid; vec < n_vec; vec += TPR) {
        const int c = vec * VN, n = (int)min((int64_t)VN, a.H - c);
        load_weight<T>(a.w, a.w_dtype, c, n, w[0]);
        // (this thread wrote these values of h itself)
        const T* src = MODE != ROWS8 && rp ? (const T*)a.h + row * a.H : xp + row * a.ldx;
        write(load_part(src + c, n), w[0], vec);
      }
    }
    if constexpr (MODE != NORM) {
      for (int64_t c = (int64_t)n_vec * VN + tid; c < a.ldq; c += TPR) a.q[row * a.ldq + c] = 0;
    }
  }
}

typedef void (*Kernel)(FwdArgs);
template <class T, int TPR, int NV> constexpr Kernel norm_k = add_rmsnorm_kernel<T, TPR, NV, NORM>;
template <class T, int TPR, int NV> constexpr Kernel norm8_k = add_rmsnorm_kernel<T, TPR, NV, NORM8>;
template <class T, int TPR, int NV> constexpr Kernel rows8_k = add_rmsnorm_kernel<T, TPR, NV, ROWS8>;

template <class T> Kernel pick_norm(int64_t H) { FROWS_PICK(T, H, norm_k); }
template <class T> Kernel pick_norm8(int64_t H) { FROWS_PICK(T, H, norm8_k); }
template <class T> Kernel pick_rows8(int64_t H) { FROWS_PICK(T, H, rows8_k); }

template <class T>
static Kernel pick(int mode, int64_t H) {
  return mode == NORM ? pick_norm<T>(H) : mode == NORM8 ? pick_norm8<T>(H) : pick_rows8<T>(H);
}

static int launch(const char* what, int dtype, int mode, const FwdArgs& a, hipStream_t s) {
  if (dtype != FORGE_DTYPE_F32 && dtype != FORGE_DTYPE_F16 && dtype != FORGE_DTYPE_BF16)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  if (a.w && a.w_dtype != FORGE_DTYPE_F32 && a.w_dtype != FORGE_DTYPE_F16 && a.w_dtype != FORGE_DTYPE_BF16)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: weight dtype %d", what, a.w_dtype);
  if (a.rows < 0 || a.H < 0 || a.H > (int64_t(1) << 30)) return forge_set_error(FORGE_ERR_INVALID, "%s: sizes", what);
  if (a.ldx < a.H || (a.res && a.ldr < a.H)) return forge_set_error(FORGE_ERR_INVALID, "%s: row pitch below %lld", what, (long long)a.H);
  if (mode != NORM && (a.ldq < a.H || a.ldq % 16 || !aligned16(a.q)))
    return forge_set_error(FORGE_ERR_INVALID, "%s: 8-bit rows need a pitch that is a multiple of 16, and 16-byte alignment", what);
  if (a.rows == 0 || a.H == 0) return FORGE_OK;
  if (!a.x || (mode == NORM ? !a.y : !a.q || !a.scale)) return forge_set_error(FORGE_ERR_INVALID, "%s: an array is NULL", what);
  const Kernel k = dtype == FORGE_DTYPE_F32 ? pick<float>(mode, a.H)
                   : dtype == FORGE_DTYPE_F16 ? pick<fp16_t>(mode, a.H) : pick<bf16_t>(mode, a.H);
  const int64_t nv = (a.H * (int64_t)dtype_size(dtype) + 15) / 16, rpb = nv <= 128 ? 4 : 1;
  const int64_t blocks = (a.rows + rpb - 1) / rpb;
  k<<<(unsigned)(blocks < 2048 ? blocks : 2048), 256, 0, s>>>(a);
  FORGE_CHECK_LAUNCH();
  return FORGE_OK;
}

}  // namespace frows

using namespace frows;

static bool narrow(int dtype) { return dtype == FORGE_DTYPE_F16 || dtype == FORGE_DTYPE_BF16; }

static FwdArgs norm_args(int w_dtype, const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                         void* h, int64_t rows, int64_t H, double eps, double offset) {
  FwdArgs a = {};
  a.x = x;
  a.ldx = ldx;
  a.res = residual;
  a.ldr = ldr;
  a.w = weight;
  a.w_dtype = w_dtype;
  a.h = h;
  a.rows = rows;
  a.H = H;
  a.eps = (float)eps;
  a.offset = (float)offset;
  return a;
}

extern "C" int forge_add_rmsnorm_fwd(int dtype, int w_dtype, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                     const void* weight, void* h, void* y, float* rstd, int64_t rows, int64_t H, double eps,
                                     double offset, void* stream) {
  FwdArgs a = norm_args(w_dtype, x, ldx, residual, ldr, weight, h, rows, H, eps, offset);
  a.y = y;
  a.rstd = rstd;
  if (rows > 0 && H > 0 && (!weight || (residual && !h))) return forge_set_error(FORGE_ERR_INVALID, "add_rmsnorm: an array is NULL");
  return launch("add_rmsnorm", dtype, NORM, a, (hipStream_t)stream);
}

extern "C" int forge_add_rmsnorm_int8(int dtype, int w_dtype, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                      const void* weight, void* h, int8_t* q, int64_t ldq, float* scale, int64_t rows,
                                      int64_t H, double eps, double offset, void* stream) {
  FwdArgs a = norm_args(w_dtype, x, ldx, residual, ldr, weight, h, rows, H, eps, offset);
  a.q = q;
  a.ldq = ldq;
  a.scale = scale;
  a.exact = narrow(dtype) && narrow(w_dtype) && offset == 0.0;
  if (rows > 0 && H > 0 && (!weight || (residual && !h))) return forge_set_error(FORGE_ERR_INVALID, "add_rmsnorm: an array is NULL");
  return launch("add_rmsnorm", dtype, NORM8, a, (hipStream_t)stream);
}

extern "C" int forge_quantize_rows(int dtype, const void* x, int64_t ldx, const float* col_scale, int8_t* q, int64_t ldq,
                                   float* scale, int64_t rows, int64_t H, void* stream) {
  FwdArgs a = {};
  a.x = x;
  a.ldx = ldx;
  a.w = col_scale;
  a.w_dtype = FORGE_DTYPE_F32;
  a.q = q;
  a.ldq = ldq;
  a.scale = scale;
  a.rows = rows;
  a.H = H;
  a.exact = col_scale == nullptr;
  return launch("quantize_rows", dtype, ROWS8, a, (hipStream_t)stream);
}
