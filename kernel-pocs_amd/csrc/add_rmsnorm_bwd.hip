// Backward of the RMS norm with the residual's addition:
//   g = dy (w + offset),  d = dh + rstd (g - h rstd (rstd mean(g h)))   (x's and the residual's)
//   dw = sum over rows of dy h rstd
// (multiplied in this order: rstd^3 itself is infinite for rows of 1e-13, and a
// subnormal for those of 1e13 and more)
// with dh the gradient that reaches h by the residual stream.  Reads dy, dh and h
// and writes d once.  A workgroup adds its rows' dw in registers (thread t its
// own columns) and writes one partial row; a second launch adds those in order.
// Bound by HBM: 16-bit [8192, 4096] 46 us (5.8 TB/s) and 4 for the partial rows.
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
  float* part;                   // [blocks][ld_part]
  int64_t ld_part;
  int64_t rows, H;
  float offset;
};

template <class T, int TPR, int NV, bool DW, bool DH>
__global__ __launch_bounds__(threads_of<TPR>) void add_rmsnorm_bwd_kernel(BwdArgs a) {
  constexpr int VN = V<T>, RPB = rows_per_block<TPR>, N = NV ? NV : 1;
  __shared__ float sums[2][threads_of<TPR> / 64];
  __shared__ float cols[TPR == 64 && DW ? 4 * 64 * N * VN : 1];
  const int tid = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int n_vec = (int)((a.H + VN - 1) / VN);
  const float inv_h = 1.f / (float)a.H;
  float w[N][VN], dw[N][VN];
  auto load_w = [&](int c, float (&o)[VN]) {
    load_weight<T>(a.w, a.w_dtype, c, (int)min((int64_t)VN, a.H - c), o);
#pragma unroll
    for (int i = 0; i < VN; ++i) o[i] += a.offset;
  };
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int vec = tid + j * TPR;
    if (NV > 0 && vec < n_vec) load_w(vec * VN, w[j]);
#pragma unroll
    for (int i = 0; i < VN; ++i) dw[j][i] = 0.f;
  }
  struct Set {
    Vec<T> h[N], dy[N], dh[N];
    float rstd;
  } sets[2];
  auto fetch = [&](int64_t row, Set& s) {
    row = min(row, a.rows - 1);
    s.rstd = a.rstd[row];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (tid + j * TPR) * VN;
      s.h[j] = load_held((const T*)a.h + row * a.ldh, c, a.H);
      s.dy[j] = load_held((const T*)a.dy + row * a.lddy, c, a.H);
      if constexpr (DH) s.dh[j] = load_held((const T*)a.dh + row * a.lddh, c, a.H);
      else s.dh[j].clear();
    }
  };
  bool started = false;  // NV = 0: this workgroup's partial row has been written
  auto work = [&](int64_t row, Set& s, int flip) __attribute__((always_inline)) {
    const bool on = row < a.rows;
    float dot = 0.f;
    auto add_dot = [&](const Vec<T>& x, const Vec<T>& y, const float (&wv)[VN]) {
#pragma unroll
      for (int i = 0; i < VN; ++i) dot += y.get(i) * wv[i] * x.get(i);
    };
    const T* hp = (const T*)a.h + row * a.ldh;
    const T* yp = (const T*)a.dy + row * a.lddy;
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (on && tid + j * TPR < n_vec) {
          const int n = (int)min((int64_t)VN, a.H - (tid + j * TPR) * VN);
          fit(s.h[j], n);
          fit(s.dy[j], n);
          if constexpr (DH) fit(s.dh[j], n);
          add_dot(s.h[j], s.dy[j], w[j]);
        }
    } else if (on) {
      for (int vec = tid; vec < n_vec; vec += TPR) {
        const int c = vec * VN, n = (int)min((int64_t)VN, a.H - c);
        load_w(c, w[0]);
        add_dot(load_part(hp + c, n), load_part(yp + c, n), w[0]);
      }
    }
    dot = row_sum<TPR>(dot, sums[flip]);
    if (!on) return;
    const float rstd = NV > 0 ? s.rstd : a.rstd[row], k = rstd * (rstd * dot * inv_h);
    auto finish = [&](const Vec<T>& x, const Vec<T>& y, const Vec<T>& g, const float (&wv)[VN], int vec) {
      Vec<T> d;
      float f[VN];
#pragma unroll
      for (int i = 0; i < VN; ++i) f[i] = g.get(i) + rstd * (y.get(i) * wv[i] - x.get(i) * k);
      d.set(f);
      const int c = vec * VN;
      store_part((T*)a.d + row * a.H + c, d, (int)min((int64_t)VN, a.H - c));
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int vec = tid + j * TPR;
        if (vec < n_vec) {
          s.h[j].keep();
          s.dy[j].keep();
          finish(s.h[j], s.dy[j], s.dh[j], w[j], vec);
          if constexpr (DW)
#pragma unroll
            for (int i = 0; i < VN; ++i) dw[j][i] += s.dy[j].get(i) * (s.h[j].get(i) * rstd);
        }
      }
    } else {
      for (int vec = tid; vec < n_vec; vec += TPR) {
        const int c = vec * VN, n = (int)min((int64_t)VN, a.H - c);
        load_w(c, w[0]);
        Vec<T> g;
        g.clear();
        if constexpr (DH) g = load_part((const T*)a.dh + row * a.lddh + c, n);
        const Vec<T> x = load_part(hp + c, n), y = load_part(yp + c, n);
        finish(x, y, g, w[0], vec);
        if constexpr (DW) {  // (this thread's own columns of the workgroup's partial row)
          float* p = a.part + blockIdx.x * a.ld_part + c;
#pragma unroll
          for (int i = 0; i < VN; ++i)
            if (i < n) {
              const float t = y.get(i) * (x.get(i) * rstd);
              p[i] = started ? p[i] + t : t;
            }
        }
      }
      started = true;
    }
  };
  // (every thread of a workgroup goes through the same rounds)
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t first = (int64_t)blockIdx.x * RPB;
  if constexpr (NV > 0) {  // the next row's loads are in flight while a row is worked on
    fetch(first + slot, sets[0]);
    for (; first < a.rows; first += 2 * step) {
      fetch(first + step + slot, sets[1]);
      work(first + slot, sets[0], 0);
      if (first + step >= a.rows) break;
      fetch(first + 2 * step + slot, sets[0]);
      work(first + step + slot, sets[1], 1);
    }
  } else {
    for (int flip = 0; first < a.rows; first += step, flip ^= 1) work(first + slot, sets[0], flip);
  }
  if constexpr (DW && NV > 0) {
    float* part = a.part + blockIdx.x * a.ld_part;
    if constexpr (TPR == 64) {  // the four waves' sums, in wave order
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
      for (int j = 0; j < N; ++j) {
        const int c = (tid + j * TPR) * VN;
#pragma unroll
        for (int i = 0; i < VN; i += 4)  // (the pitch is a multiple of 4)
          if (c + i < a.H) *reinterpret_cast<float4*>(part + c + i) = make_float4(dw[j][i], dw[j][i + 1], dw[j][i + 2], dw[j][i + 3]);
      }
    }
  }
}

// dw[c] = sum of the partial rows.  32 columns a workgroup, 4 a thread: 32 groups of
// 8 threads add consecutive blocks of rows, and one of them the groups' sums, in
// order.
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* part, int64_t ld, int n, int64_t H, void* dw, int w_dtype) {
  __shared__ float4 red[32][8];
  const int c4 = threadIdx.x % 8, g = threadIdx.x / 8;
  const int64_t col = (int64_t)blockIdx.x * 32 + 4 * c4;
  const int per = (n + 31) / 32, lo = g * per, hi = min(n, lo + per);
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < H) {
#pragma unroll 8
    for (int r = lo; r < hi; ++r) {
      const float4 v = *reinterpret_cast<const float4*>(part + r * ld + col);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
  }
  red[g][c4] = s;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  if (c >= H) return;
  const float* f = reinterpret_cast<const float*>(&red[0][0]) + threadIdx.x;
  float t = f[0];
#pragma unroll
  for (int k = 1; k < 32; ++k) t += f[32 * k];
  if (w_dtype == FORGE_DTYPE_F32) ((float*)dw)[c] = t;
  else if (w_dtype == FORGE_DTYPE_F16) ((fp16_t*)dw)[c] = (fp16_t)t;
  else ((bf16_t*)dw)[c] = (bf16_t)t;
}

typedef void (*BwdKernel)(BwdArgs);
template <class T, int TPR, int NV, bool DW, bool DH> constexpr BwdKernel bwd_k = add_rmsnorm_bwd_kernel<T, TPR, NV, DW, DH>;
template <class T, bool DW, bool DH> static BwdKernel pick_one(int64_t H) { FROWS_PICK(T, H, bwd_k, DW, DH); }
template <class T> static BwdKernel pick_bwd(int64_t H, bool dw, bool dh) {
  return dw ? (dh ? pick_one<T, true, true>(H) : pick_one<T, true, false>(H)) : dh ? pick_one<T, false, true>(H) : pick_one<T, false, false>(H);
}

static int64_t part_pitch(int64_t H) { return (H + 3) / 4 * 4; }

// Workgroups: one partial row each.
static int64_t bwd_blocks(int dtype, int64_t rows, int64_t H) {
  const int at_once = rows_at_once(H, dtype_size(dtype));
  const int64_t blocks = (rows + at_once - 1) / at_once;
  return blocks < 512 ? blocks : 512;
}

}  // namespace frows

using namespace frows;

extern "C" int64_t forge_add_rmsnorm_bwd_workspace(int dtype, int64_t rows, int64_t H) {
  if (rows < 0 || H < 0 || dtype_size(dtype) == 0) return -1;
  return bwd_blocks(dtype, rows, H) * part_pitch(H) * 4;
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
  if (dw && !aligned16(work)) return forge_set_error(FORGE_ERR_INVALID, "add_rmsnorm: work is not 16-byte aligned");
  BwdArgs a = {dy, lddy, dh, lddh, h, ldh, weight, w_dtype, rstd, d, (float*)work, part_pitch(H), rows, H, (float)offset};
  const BwdKernel k = dtype == FORGE_DTYPE_F32 ? pick_bwd<float>(H, dw, dh) : dtype == FORGE_DTYPE_F16 ? pick_bwd<fp16_t>(H, dw, dh) : pick_bwd<bf16_t>(H, dw, dh);
  const int64_t blocks = bwd_blocks(dtype, rows, H);
  k<<<(unsigned)blocks, threads_for(H, dtype_size(dtype)), 0, (hipStream_t)stream>>>(a);
  FORGE_CHECK_LAUNCH();
  if (dw) {
    sum_parts_kernel<<<(unsigned)((H + 31) / 32), 256, 0, (hipStream_t)stream>>>((const float*)work, part_pitch(H), (int)blocks, H, dw, w_dtype);
    FORGE_CHECK_LAUNCH();
  }
  return FORGE_OK;
}
