// Backward of the RMS norm with the residual's addition:
//   g = dy (w + offset),  d = dh + rstd g - h rstd^3 mean(g h)   (x's and the residual's)
//   dw = sum over rows of dy h rstd
// with dh the gradient that reaches h by the residual stream.  Reads dy, dh and h
// and writes d once.  A workgroup adds its rows' dw in registers (thread t its
// own columns) and writes one partial row; a second launch adds those in order.
#include "add_rmsnorm.h"

namespace frows {

struct BwdArgs {
  const void* dy; int64_t lddy;
  const void* dh; int64_t lddh;  // or NULL
  const void* h;                 // [rows][ldh]
  int64_t ldh;
  const void* w; int w_dtype;
  const float* rstd;
  void* d;                       // [rows][H]
  float* part;                   // [blocks][H], or NULL
  int64_t rows, H;
  float offset;
};

template <class T, int TPR, int NV>
__global__ __launch_bounds__(256) void add_rmsnorm_bwd_kernel(BwdArgs a) {
  constexpr int VN = V<T>, RPB = rows_per_block<TPR>, N = NV ? NV : 1;
  __shared__ float sums[2][4];
  __shared__ float cols[TPR == 64 ? 4 * 64 * N * VN : 1];
  const int tid = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int n_vec = (int)((a.H + VN - 1) / VN);
  const float inv_h = 1.f / (float)a.H;
  float w[N][VN], dw[N][VN];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (tid + j * TPR) * VN;
    load_weight<T>(a.w, a.w_dtype, c, (int)(a.H - c), w[j]);
#pragma unroll
    for (int i = 0; i < VN; ++i) dw[j][i] = 0.f;
  }
  int flip = 0;
  for (int64_t first = (int64_t)blockIdx.x * RPB; first < a.rows; first += (int64_t)gridDim.x * RPB, flip ^= 1) {
    const int64_t row = first + slot;
    const bool on = row < a.rows;
    const float rstd = on ? a.rstd[row] : 0.f;
    Vec16<T> h[N], dy[N], dh[N];
    const T* hp = (const T*)a.h + row * a.ldh;
    const T* yp = (const T*)a.dy + row * a.lddy;
    const T* sp = (const T*)a.dh + row * a.lddh;
    float dot = 0.f;
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int vec = tid + j * TPR, c = vec * VN, n = (int)min((int64_t)VN, a.H - c);
        if (on && vec < n_vec) {
          h[j] = load_part(hp + c, n);
          dy[j] = load_part(yp + c, n);
          if (a.dh) dh[j] = load_part(sp + c, n);
          else dh[j].raw = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < VN; ++i) dot += to_f32(dy[j].v[i]) * (w[j][i] + a.offset) * to_f32(h[j].v[i]);
        }
      }
    } else if (on) {
      for (int vec = tid; vec < n_vec; vec += TPR) {
        const int c = vec * VN, n = (int)min((int64_t)VN, a.H - c);
        load_weight<T>(a.w, a.w_dtype, c, n, w[0]);
        const Vec16<T> x = load_part(hp + c, n), y = load_part(yp + c, n);
#pragma unroll
        for (int i = 0; i < VN; ++i) dot += to_f32(y.v[i]) * (w[0][i] + a.offset) * to_f32(x.v[i]);
      }
    }
    dot = row_sum<TPR>(dot, sums[flip]);
    const float k = rstd * rstd * rstd * dot * inv_h;
    auto finish = [&](const Vec16<T>& x, const Vec16<T>& y, const Vec16<T>& s, const float (&wv)[VN], int vec) {
      Vec16<T> d;
#pragma unroll
      for (int i = 0; i < VN; ++i)
        d.v[i] = from_f32<T>(to_f32(s.v[i]) + (rstd * (to_f32(y.v[i]) * (wv[i] + a.offset)) - to_f32(x.v[i]) * k));
      const int c = vec * VN;
      store_part((T*)a.d + row * a.H + c, d, (int)min((int64_t)VN, a.H - c));
    };
    if (!on) continue;
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int vec = tid + j * TPR;
        if (vec < n_vec) {
          finish(h[j], dy[j], dh[j], w[j], vec);
#pragma unroll
          for (int i = 0; i < VN; ++i) dw[j][i] += to_f32(dy[j].v[i]) * (to_f32(h[j].v[i]) * rstd);
        }
      }
    } else {
      for (int vec = tid; vec < n_vec; vec += TPR) {
        const int c = vec * VN, n = (int)min((int64_t)VN, a.H - c);
        load_weight<T>(a.w, a.w_dtype, c, n, w[0]);
        Vec16<T> s;
        s.raw = make_uint4(0, 0, 0, 0);
        if (a.dh) s = load_part(sp + c, n);
        const Vec16<T> x = load_part(hp + c, n), y = load_part(yp + c, n);
        finish(x, y, s, w[0], vec);
        if (a.part) {  // (this thread's own columns of the workgroup's partial row)
          float* p = a.part + blockIdx.x * a.H + c;
#pragma unroll
          for (int i = 0; i < VN; ++i)
            if (i < n) {
              const float t = to_f32(y.v[i]) * (to_f32(x.v[i]) * rstd);
              p[i] = first == (int64_t)blockIdx.x * RPB ? t : p[i] + t;
            }
        }
      }
    }
  }
  if (!a.part || NV == 0) return;
  float* part = a.part + blockIdx.x * a.H;
  if constexpr (TPR == 64) {  // the four waves' sums, in wave order
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < VN; ++i) cols[slot * 64 * N * VN + (tid + j * 64) * VN + i] = dw[j][i];
    __syncthreads();
    for (int c = threadIdx.x; c < a.H; c += 256) {
      float s = cols[c];
#pragma unroll
      for (int k = 1; k < 4; ++k) s += cols[k * 64 * N * VN + c];
      part[c] = s;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        const int c = (tid + j * TPR) * VN + i;
        if (c < a.H) part[c] = dw[j][i];
      }
  }
}

// dw[c] = sum of the partial rows: 32 columns a workgroup, 8 groups of threads
// add consecutive blocks of rows, one of them the groups' sums, in order.
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* part, int n, int64_t H, void* dw, int w_dtype) {
  __shared__ float red[8][32];
  const int c = threadIdx.x % 32, g = threadIdx.x / 32;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  const int per = (n + 7) / 8, lo = g * per, hi = min(n, lo + per);
  float s = 0.f;
  if (col < H)
    for (int r = lo; r < hi; ++r) s += part[r * H + col];
  red[g][c] = s;
  __syncthreads();
  if (g == 0 && col < H) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][c];
    if (w_dtype == FORGE_DTYPE_F32) ((float*)dw)[col] = s;
    else if (w_dtype == FORGE_DTYPE_F16) ((fp16_t*)dw)[col] = (fp16_t)s;
    else ((bf16_t*)dw)[col] = (bf16_t)s;
  }
}

typedef void (*BwdKernel)(BwdArgs);
template <class T, int TPR, int NV> constexpr BwdKernel bwd_k = add_rmsnorm_bwd_kernel<T, TPR, NV>;
template <class T> BwdKernel pick_bwd(int64_t H) { FROWS_PICK(T, H, bwd_k); }

// Workgroups: one partial row each.
static int64_t bwd_blocks(int dtype, int64_t rows, int64_t H) {
  const int64_t nv = (H * (int64_t)dtype_size(dtype) + 15) / 16, rpb = nv <= 128 ? 4 : 1;
  const int64_t blocks = (rows + rpb - 1) / rpb;
  return blocks < 512 ? blocks : 512;
}

}  // namespace frows

using namespace frows;

extern "C" int64_t forge_add_rmsnorm_bwd_workspace(int dtype, int64_t rows, int64_t H) {
  if (rows < 0 || H < 0 || dtype_size(dtype) == 0) return -1;
  return bwd_blocks(dtype, rows, H) * H * 4;
}

extern "C" int forge_add_rmsnorm_bwd(int dtype, int w_dtype, const void* dy, int64_t lddy, const void* dh, int64_t lddh,
                                     const void* h, int64_t ldh, const void* weight, const float* rstd, void* d, void* dw,
                                     void* work, int64_t rows, int64_t H, double offset, void* stream) {
  if (dtype != FORGE_DTYPE_F32 && dtype != FORGE_DTYPE_F16 && dtype != FORGE_DTYPE_BF16)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "add_rmsnorm: dtype %d", dtype);
  if (w_dtype != FORGE_DTYPE_F32 && w_dtype != FORGE_DTYPE_F16 && w_dtype != FORGE_DTYPE_BF16)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "add_rmsnorm: weight dtype %d", w_dtype);
  if (rows < 0 || H < 0 || H > (int64_t(1) << 30)) return forge_set_error(FORGE_ERR_INVALID, "add_rmsnorm: sizes");
  if (lddy < H || ldh < H || (dh && lddh < H)) return forge_set_error(FORGE_ERR_INVALID, "add_rmsnorm: row pitch below %lld", (long long)H);
  if (rows == 0 || H == 0) return FORGE_OK;  // (the caller clears dw)
  if (!dy || !h || !weight || !rstd || !d || (dw && !work)) return forge_set_error(FORGE_ERR_INVALID, "add_rmsnorm: an array is NULL");
  BwdArgs a = {dy, lddy, dh, lddh, h, ldh, weight, w_dtype, rstd, d, dw ? (float*)work : nullptr, rows, H, (float)offset};
  const BwdKernel k = dtype == FORGE_DTYPE_F32 ? pick_bwd<float>(H) : dtype == FORGE_DTYPE_F16 ? pick_bwd<fp16_t>(H) : pick_bwd<bf16_t>(H);
  const int64_t blocks = bwd_blocks(dtype, rows, H);
  k<<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>(a);
  FORGE_CHECK_LAUNCH();
  if (dw) {
    sum_parts_kernel<<<(unsigned)((H + 31) / 32), 256, 0, (hipStream_t)stream>>>((const float*)work, (int)blocks, H, dw, w_dtype);
    FORGE_CHECK_LAUNCH();
  }
  return FORGE_OK;
}
