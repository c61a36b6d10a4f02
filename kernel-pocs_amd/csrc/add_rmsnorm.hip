// RMS norm with the residual's addition, and rows in 8 bits with one scale each.
//
//   h = round(x + residual)                       (stored: the residual stream)
//   y = round(h rstd (w + offset)),  rstd = 1 / sqrt(mean h^2 + eps)
//   or, in 8 bits, with t = h (w + offset) and a = max |t| of the row:
//   q = round_half_even(127 t / a),  scale = a rstd / 127:  y = q scale
// The integers do not depend on rstd, and both sums of a row are taken in one
// pass.  Rows as they are (no norm): t = x, or x times a scale a column.
//
// The integers are those of exact arithmetic.  127 / a lies between two neighbours
// below and above its value in fp32, t times each is rounded to an integer once (an fma
// with 1.5 2^23, whose last byte it is), and as rounding keeps the order the
// integer is that of t's exact quotient where both agree.  They differ where a border
// between two integers lies within some 2^-23 of the quotient: those vectors are
// divided again, in 64 bits.  t of two 16-bit factors is exact in fp32; otherwise the
// largest is found in 64 bits and the two are 6 steps off, for the roundings of t.
//
// Bound by HBM: x and the residual are read once, h and y written once.  16-bit [8192,
// 4096]: 45 us (5.9 TB/s), to 8 bits 45 (5.2).  16-bit rows of [8192, 14336] to 8 bits
// 84 us (4.2 TB/s): no row's bytes are written before all of it has been read.
#include "add_rmsnorm.h"

namespace frows {

struct FwdArgs {
  const void* x; int64_t ldx;
  const void* res; int64_t ldr;  // or NULL
  const void* w; int w_dtype;
  void* h;                       // [rows][H], or NULL where there is no residual
  void* y;                       // [rows][H]
  int8_t* q; int64_t ldq;        // [rows][ldq], zeros from H on
  float* scale;                  // [rows]
  float* rstd;                   // [rows], or NULL
  int64_t rows, H;
  float eps, offset;
};

// What becomes of a row: its norm, its norm in 8 bits (the products exact in fp32, or
// not), the row itself in 8 bits, or times a scale a column.
enum Mode { NORM, NORM8, NORM8_WIDE, ROWS8, ROWS8_SCALED };

// The integers of V values of a row with factors w, as bytes; below and above: of 127 / a.
template <class T, bool UNIT>
__device__ __forceinline__ void quantize(const Vec<T>& v, const float* w, double offset, float below, float above, double a,
                                         bool tiny, uint32_t (&word)[V<T> / 4]) {
  uint32_t k[V<T>], differ = tiny;
#pragma unroll
  for (int i = 0; i < V<T>; ++i) {
    const float t = UNIT ? v.get(i) : v.get(i) * (w[i] + (float)offset);
    k[i] = __float_as_uint(__builtin_fmaf(t, below, 0x1.8p23f));
    differ |= k[i] ^ __float_as_uint(__builtin_fmaf(t, above, 0x1.8p23f));
  }
  if (differ) {
#pragma unroll
    for (int i = 0; i < V<T>; ++i) {
      const double t = UNIT ? (double)v.get(i) : (double)v.get(i) * ((double)w[i] + offset);
      k[i] = (uint32_t)(int)rint(127.0 * t / a);
    }
  }
#pragma unroll
  for (int i = 0; i < V<T>; i += 4)
    word[i / 4] = __builtin_amdgcn_perm(k[i + 1], k[i], 0x0c0c0400) | __builtin_amdgcn_perm(k[i + 3], k[i + 2], 0x04000c0c);
}

template <class T, int TPR, int NV, int MODE, bool RES>
__global__ __launch_bounds__(threads_of<TPR>) void add_rmsnorm_kernel(FwdArgs a) {
  constexpr int VN = V<T>, RPB = rows_per_block<TPR>, N = NV ? NV : 1;
  constexpr bool SUMS = MODE == NORM || MODE == NORM8 || MODE == NORM8_WIDE, EIGHT = MODE != NORM;
  constexpr bool WIDE = MODE == NORM8_WIDE || MODE == ROWS8_SCALED, UNIT = MODE == ROWS8;
  constexpr bool HELD = !UNIT && NV > 0;  // a thread's weights
  constexpr int WAVES = threads_of<TPR> / 64;
  __shared__ float sums[2][WAVES];
  __shared__ uint32_t tops[2][WAVES];
  __shared__ double tops64[2][WAVES];
  const int tid = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int n_vec = (int)((a.H + VN - 1) / VN);
  const T* xp = (const T*)a.x;
  const T* rp = (const T*)a.res;
  // the factors of t: weight + offset, of which WIDE adds the offset in 64 bits
  const float add = WIDE ? 0.f : a.offset;
  const double add64 = WIDE ? (double)a.offset : 0.0;
  float w[HELD ? N : 1][VN];
  auto load_w = [&](int c, float (&o)[VN]) {
    load_weight<T>(a.w, a.w_dtype, c, (int)min((int64_t)VN, a.H - c), o);
#pragma unroll
    for (int i = 0; i < VN; ++i) o[i] += add;
  };
  if constexpr (HELD) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int vec = tid + j * TPR;
      if (vec < n_vec) load_w(vec * VN, w[j]);
    }
  }
  Vec<T> x[2][N], r[2][N];
  auto fetch = [&](int64_t row, int set) {
    row = min(row, a.rows - 1);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (tid + j * TPR) * VN;
      x[set][j] = load_held(xp + row * a.ldx, c, a.H);
      if constexpr (RES) r[set][j] = load_held(rp + row * a.ldr, c, a.H);
    }
  };
  auto sum = [&](const Vec<T>& u, const Vec<T>& v) {
    Vec<T> h;
    float f[VN];
#pragma unroll
    for (int i = 0; i < VN; ++i) f[i] = u.get(i) + v.get(i);
    h.set(f);
    return h;
  };

  auto work = [&](int64_t row, int set, int flip) __attribute__((always_inline)) {
    float ss = 0.f;
    uint32_t top = 0;
    double top64 = 0.0;
    auto see = [&](const Vec<T>& v, const float* wv) {
      if constexpr (UNIT && sizeof(T) == 2) {  // magnitudes of two values at once
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top),
                                                                       __builtin_bit_cast(u16x2, v.w[i] & 0x7fff7fffu)));
        return;
      }
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        const float f = v.get(i);
        if (SUMS) ss += f * f;
        if (EIGHT) top = max(top, __float_as_uint(UNIT ? f : f * (wv[i] + (float)add64)) & 0x7fffffffu);
        if (WIDE) top64 = fmax(top64, fabs((double)f * ((double)wv[i] + add64)));
      }
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int vec = tid + j * TPR;
        if (vec < n_vec) {
          const int n = (int)min((int64_t)VN, a.H - vec * VN);
          fit(x[set][j], n);
          if constexpr (RES) {
            fit(r[set][j], n);
            x[set][j] = sum(x[set][j], r[set][j]);
            store_part((T*)a.h + row * a.H + vec * VN, x[set][j], n);
          }
          see(x[set][j], w[HELD ? j : 0]);
        }
      }
    } else {
      for (int vec = tid; vec < n_vec; vec += TPR) {
        const int c = vec * VN, n = (int)min((int64_t)VN, a.H - c);
        Vec<T> v = load_part(xp + row * a.ldx + c, n);
        if (RES) {
          v = sum(v, load_part(rp + row * a.ldr + c, n));
          store_part((T*)a.h + row * a.H + c, v, n);
        }
        if (!UNIT) load_w(c, w[0]);
        see(v, w[0]);
      }
    }
    float rstd = 1.f;
    if constexpr (EIGHT) {
      if constexpr (UNIT && sizeof(T) == 2) {  // (their order is that of what they stand for)
        Vec<T> m;
        m.w[0] = max(top & 0xffffu, top >> 16);
        top = __float_as_uint(m.get(0));
      }
      top = over_wave(top, [](uint32_t p, uint32_t q) { return max(p, q); });
      if constexpr (WIDE) top64 = over_wave(top64, [](double p, double q) { return fmax(p, q); });
      if constexpr (TPR > 64) {
        if (threadIdx.x % 64 == 0) {
          tops[flip][threadIdx.x / 64] = top;
          if (WIDE) tops64[flip][threadIdx.x / 64] = top64;
        }
        if (!SUMS) __syncthreads();
      }
    }
    if constexpr (SUMS) {
      ss = row_sum<TPR>(ss, sums[flip]);
      rstd = rsqrtf(ss / (float)a.H + a.eps);
      if (tid == 0 && a.rstd) a.rstd[row] = rstd;
    }
    float below = 0.f, above = 0.f;
    bool tiny = false, bad = false;
    if constexpr (EIGHT) {
      if constexpr (TPR > 64) {
#pragma unroll
        for (int k = 0; k < TPR / 64; ++k) {
          top = max(top, tops[flip][k]);
          if (WIDE) top64 = fmax(top64, tops64[flip][k]);
        }
      }
      if (!WIDE) top64 = (double)__uint_as_float(top);
      // infinities and NaN: the row's scale is NaN, and so is all that is computed of it
      bad = top >= 0x7f800000u;
      tiny = top64 < 1e-30;
      if (!tiny && !bad) {
        const uint32_t inv = __float_as_uint(127.f / (float)top64);
        below = __uint_as_float(inv - (WIDE ? 6 : 1));
        above = __uint_as_float(inv + (WIDE ? 6 : 1));
      }
      // (a rstd may pass fp32's range where a rstd / 127 does not)
      if (tid == 0)
        a.scale[row] = bad ? __builtin_nanf("") : SUMS ? (float)(top64 * (double)rstd / 127.0) : (float)top64 / 127.f;
    }
    auto write = [&](const Vec<T>& v, const float* wv, int vec) {
      const int c = vec * VN;
      if constexpr (!EIGHT) {
        Vec<T> y;
        float f[VN];
#pragma unroll
        for (int i = 0; i < VN; ++i) f[i] = v.get(i) * rstd * wv[i];
        y.set(f);
        store_part((T*)a.y + row * a.H + c, y, (int)min((int64_t)VN, a.H - c));
      } else {
        uint32_t word[VN / 4];
        if (bad || top64 == 0.0) {
#pragma unroll
          for (int k = 0; k < VN / 4; ++k) word[k] = 0;
        } else {
          // (values behind the row's end are zeros)
          quantize<T, UNIT>(v, wv, add64, below, above, top64, tiny, word);
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
        if (vec < n_vec) {
          x[set][j].keep();
          write(x[set][j], w[HELD ? j : 0], vec);
        }
      }
    } else {
      for (int vec = tid; vec < n_vec; vec += TPR) {
        const int c = vec * VN, n = (int)min((int64_t)VN, a.H - c);
        if (!UNIT) load_w(c, w[0]);
        // (this thread wrote these values of h itself)
        const T* src = RES ? (const T*)a.h + row * a.H : xp + row * a.ldx;
        write(load_part(src + c, n), w[0], vec);
      }
    }
    if constexpr (EIGHT) {
      for (int64_t c = (int64_t)n_vec * VN + tid; c < a.ldq; c += TPR) a.q[row * a.ldq + c] = 0;
    }
  };

  // (every thread of a workgroup goes through the same rounds: sums over a row have barriers)
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + slot;
  if constexpr (NV > 0) {  // the next row's loads are in flight while a row is worked on
    fetch(row, 0);
    for (; row < a.rows; row += 2 * step) {
      fetch(row + step, 1);
      work(row, 0, 0);
      if (row + step >= a.rows) break;
      fetch(row + 2 * step, 0);
      work(row + step, 1, 1);
    }
  } else {
    for (int flip = 0; row < a.rows; row += step, flip ^= 1) work(row, 0, flip);
  }
}

typedef void (*Kernel)(FwdArgs);
template <class T, int TPR, int NV, int MODE, bool RES> constexpr Kernel fwd_k = add_rmsnorm_kernel<T, TPR, NV, MODE, RES>;
template <class T, int MODE, bool RES> static Kernel pick_mode(int64_t H) { FROWS_PICK(T, H, fwd_k, MODE, RES); }

template <class T>
static Kernel pick(int mode, int64_t H, bool res) {
  switch (mode) {
    case NORM: return res ? pick_mode<T, NORM, true>(H) : pick_mode<T, NORM, false>(H);
    case NORM8:
      if constexpr (sizeof(T) == 2) return res ? pick_mode<T, NORM8, true>(H) : pick_mode<T, NORM8, false>(H);
    case NORM8_WIDE: return res ? pick_mode<T, NORM8_WIDE, true>(H) : pick_mode<T, NORM8_WIDE, false>(H);
    case ROWS8: return pick_mode<T, ROWS8, false>(H);
    default: return pick_mode<T, ROWS8_SCALED, false>(H);
  }
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
  const bool res = a.res != nullptr;
  const Kernel k = dtype == FORGE_DTYPE_F32 ? pick<float>(mode, a.H, res)
                   : dtype == FORGE_DTYPE_F16 ? pick<fp16_t>(mode, a.H, res) : pick<bf16_t>(mode, a.H, res);
  const int size = dtype_size(dtype), at_once = rows_at_once(a.H, size);
  const int64_t blocks = (a.rows + at_once - 1) / at_once;
  // Workgroups that stay while the rows go by, the next row of each in flight: few where
  // a row is long or gives much to do, more where its loads are most of it (16-bit
  // [8192, 4096]: norm 51 us by 2048, 48 by 1024, 45 by 512; a row times scales 27, 27, 32;
  // a row as it is 27, 30, 36; [8192, 14336]: 86, 84, 84).
  const int threads = threads_for(a.H, size), most = at_once > 1 ? 2048 : threads > 256 || mode == NORM ? 512 : mode == ROWS8 ? 2048 : 1024;
  k<<<(unsigned)(blocks < most ? blocks : most), threads, 0, s>>>(a);
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
  // (a product of two 16-bit values is exact in fp32)
  const int mode = narrow(dtype) && narrow(w_dtype) && offset == 0.0 ? NORM8 : NORM8_WIDE;
  if (rows > 0 && H > 0 && (!weight || (residual && !h))) return forge_set_error(FORGE_ERR_INVALID, "add_rmsnorm: an array is NULL");
  return launch("add_rmsnorm", dtype, mode, a, (hipStream_t)stream);
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
  return launch("quantize_rows", dtype, col_scale ? ROWS8_SCALED : ROWS8, a, (hipStream_t)stream);
}
