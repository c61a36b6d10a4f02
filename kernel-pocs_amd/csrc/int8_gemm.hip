// Products of 8-bit integers with a scale for each token and each channel:
//   C[m, n] = (sum_k a[m, k] b[n, k]) row_scale[m] col_scale[n] + bias[n]
// a [M][K] and b [N][K], K-contiguous with pitches that are multiples of 16
// bytes and zeros from K to the next multiple of 16.  The sum is exact in 32-bit
// integers; C is formed of it in fp32 (scale_i8) and rounded to fp32, bf16 or fp16.
//
// The engines are those of the 16-bit products (gemm_w4.h, gemm_core.h,
// gemm_rows.hip), which see two values as one 16-bit word: the matrix
// instructions take as many bytes a lane in the same time, so a product runs in
// the time of a 16-bit one of half the K, less what the epilogue adds.  [8192, 4096], K =
// 14336 340 us (2830 TOP/s), [8192, 14336], K = 4096 390 (2470: its epilogue converts and writes
// 235 MB); 16 rows by 28672, K = 4096 26 us (weights at 4.5 TB/s).
#include "gemm_launch.h"

namespace fgemm {

int launch_rows_i8(int out_dtype, const GemmArgs& a, hipStream_t s);

template <class O, int EPI>
static int launch_i8_big(const GemmArgs& a, hipStream_t s) {
  const int64_t tm = (a.M + 255) / 256, tn = (a.N + 255) / 256;
  if (tm * tn > 0x7fffffffLL) return forge_set_error(FORGE_ERR_INVALID, "int8_gemm: too many tiles");
  const dim3 grid((unsigned)(tm * tn), 1, (unsigned)a.split_k);
  if (a.ep.vec_ok) gemm_w4_kernel<I8<O>, B_SINGLE, EPI, true><<<grid, 256, 0, s>>>(a);
  else gemm_w4_kernel<I8<O>, B_SINGLE, EPI, false><<<grid, 256, 0, s>>>(a);
  FORGE_CHECK_LAUNCH();
  return FORGE_OK;
}

template <class O, int BM, int BN, int NS, int WPE>
static int launch_i8_tile(const GemmArgs& a, hipStream_t s) {
  constexpr int EPI = std::is_same_v<O, float> ? EPI_STORE_F32 : EPI_STORE_BF16;
  const int64_t tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
  if (tm * tn > 0x7fffffffLL) return forge_set_error(FORGE_ERR_INVALID, "int8_gemm: too many tiles");
  gemm_dma_kernel<I8<O>, BM, BN, 2, 2, EPI, 64, NS, false, WPE><<<dim3((unsigned)(tm * tn), 1, (unsigned)a.split_k), 256, 0, s>>>(a);
  FORGE_CHECK_LAUNCH();
  return FORGE_OK;
}

// The engine by the product's size.  Measured on MI355X, weights not cached, us:
//   rows (gemm_rows.hip): up to 32 rows; up to 64 of [4096] x K = 4096 and less, [33,
//     1024] 9.7, [64, 4096] 14.4 against 12.0 and 14.7 with 64 x 64 tiles split 4 ways;
//   256 x 256 tiles from 128 of them on: [2000, 14336], K = 4096 114, 128 x 128 tiles 184;
//   64 x 128 tiles where they fill the chip: [1000, 4096], K = 4096 34, 64 x 64 tiles 43,
//     256 x 256 49; [4000, 1024] 30 / 38 / 47;
//   64 x 64 tiles, split over K where they are few and K is long: [100, 1024], K =
//     14336 48 -> 16 in 8 parts, [128, 4096], K = 14336 50 -> 30 in 4, [100, 4096], K = 4096
//     18.8 -> 16.7; not [333, 1008], K = 2016: 10.9, 12.5 in 2.
enum Engine { ROWS, BIG, TILE_128, TILE_64 };
struct Plan {
  int engine, split;
};

static Plan plan_i8(int64_t M, int64_t N, int64_t K) {
  auto tiles = [&](int64_t bm, int64_t bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  if (M <= 32 || (M <= 64 && N <= 4096 && K <= 4096)) return {ROWS, 1};
  if (tiles(256, 256) >= 128) return {BIG, 1};
  if (tiles(64, 128) >= 256) return {TILE_128, 1};
  const int64_t t = tiles(64, 64), steps = (K + 127) / 128;
  int64_t split = steps < 32 ? 1 : 512 / t < steps / 8 ? 512 / t : steps / 8;
  return {TILE_64, (int)(split < 1 ? 1 : split > 8 ? 8 : split)};
}

static int64_t part_pitch(int64_t N) { return (N + 3) / 4 * 4; }

// C from the integers of the parts of K, whose sum is still exact.
template <class O>
__global__ __launch_bounds__(256) void join_i8_kernel(const int* parts, int64_t stride, int n, int64_t M, int64_t N, int64_t vecs,
                                                      EpiArgs ep) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / vecs, c = i % vecs * 4;
  if (m >= M) return;
  i32x4 sum = {0, 0, 0, 0};
  for (int z = 0; z < n; ++z) sum += *reinterpret_cast<const i32x4*>(parts + z * stride + m * vecs * 4 + c);
  const float row = ep.row_scale[m];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (c + q < N) ((O*)ep.c)[m * ep.ldc + c + q] = from_f32<O>(scale_i8(sum[q], row, ep.col_scale[c + q], bias_i8(ep, c + q)));
}

template <class O>
static int launch_i8(int out_dtype, const GemmArgs& a, const Plan& p, int* work, hipStream_t s) {
  constexpr int EPI = std::is_same_v<O, float> ? EPI_STORE_F32 : EPI_STORE_BF16;
  if (p.engine == ROWS) return launch_rows_i8(out_dtype, a, s);
  if (p.engine == BIG) return launch_i8_big<O, EPI>(a, s);
  if (p.engine == TILE_128) return launch_i8_tile<O, 64, 128, 3, 2>(a, s);
  if (p.split == 1) return launch_i8_tile<O, 64, 64, 3, 3>(a, s);
  GemmArgs g = a;  // the parts' integers
  g.ep.c = work;
  g.ep.ldc = part_pitch(a.N);
  g.ep.split_stride = a.M * g.ep.ldc;
  g.split_k = p.split;
  if (int e = launch_i8_tile<int, 64, 64, 3, 3>(g, s)) return e;
  const int64_t items = a.M * (g.ep.ldc / 4);
  join_i8_kernel<O><<<(unsigned)((items + 255) / 256), 256, 0, s>>>(work, g.ep.split_stride, p.split, a.M, a.N, g.ep.ldc / 4, a.ep);
  FORGE_CHECK_LAUNCH();
  return FORGE_OK;
}

}  // namespace fgemm

using namespace fgemm;

extern "C" int64_t forge_int8_gemm_workspace(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0) return -1;
  if (M == 0 || N == 0) return 0;
  const Plan p = plan_i8(M, N, (K + 15) / 16 * 16);
  return p.split > 1 ? p.split * M * part_pitch(N) * 4 : 0;
}

static int check_types(const char* what, int c_dtype, const void* bias, int bias_dtype) {
  auto known = [](int t) { return t == FORGE_DTYPE_F32 || t == FORGE_DTYPE_F16 || t == FORGE_DTYPE_BF16; };
  if (!known(c_dtype)) return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: C dtype %d", what, c_dtype);
  if (bias && !known(bias_dtype)) return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: bias dtype %d", what, bias_dtype);
  return FORGE_OK;
}

extern "C" int forge_int8_gemm_typed(const int8_t* a, int64_t lda, const float* row_scale, const int8_t* b, int64_t ldb,
                                     const float* col_scale, const void* bias, int bias_dtype, void* c, int64_t ldc,
                                     int c_dtype, int64_t M, int64_t N, int64_t K, void* work, void* stream) {
  if (M < 0 || N < 0 || K < 0 || K > (int64_t(1) << 17))
    return forge_set_error(FORGE_ERR_INVALID, "int8_gemm: sizes (K up to 2^17, where a sum fits 32 bits)");
  if (int e = check_types("int8_gemm", c_dtype, bias, bias_dtype)) return e;
  if (M == 0 || N == 0) return FORGE_OK;
  const int64_t kp = (K + 15) / 16 * 16;
  if (!row_scale || !col_scale || !c || (K > 0 && (!a || !b))) return forge_set_error(FORGE_ERR_INVALID, "int8_gemm: an array is NULL");
  if (lda < kp || ldb < kp || lda % 16 || ldb % 16 || lda >= (int64_t(1) << 22) || ldb >= (int64_t(1) << 22))
    return forge_set_error(FORGE_ERR_INVALID, "int8_gemm: pitches are multiples of 16 from K to 2^22");
  if (!aligned16(a) || !aligned16(b)) return forge_set_error(FORGE_ERR_INVALID, "int8_gemm: operands are 16-byte aligned");
  if (ldc < N) return forge_set_error(FORGE_ERR_INVALID, "int8_gemm: ldc below N");
  GemmArgs g = {};
  g.M = M;
  g.N = N;
  g.n_segs = 1;
  g.split_k = 1;
  g.segs[0].a = (const __bf16*)a;
  g.segs[0].lda = lda / 2;
  g.segs[0].b = (const __bf16*)b;
  g.segs[0].ldb = ldb / 2;
  g.segs[0].k = kp / 2;
  g.segs[0].n_hi = N;
  g.ep.c = c;
  g.ep.ldc = ldc;
  g.ep.alpha = 1.f;
  g.ep.row_scale = row_scale;
  g.ep.col_scale = col_scale;
  g.ep.bias = bias;
  g.ep.bias_dtype = bias_dtype;
  g.ep.vec_ok = aligned16(c) && ldc % 8 == 0;
  const Plan p = plan_i8(M, N, kp);
  if (p.split > 1 && (!work || !aligned16(work))) return forge_set_error(FORGE_ERR_INVALID, "int8_gemm: work is NULL or not aligned");
  const hipStream_t s = (hipStream_t)stream;
  if (c_dtype == FORGE_DTYPE_F32) return launch_i8<float>(c_dtype, g, p, (int*)work, s);
  if (c_dtype == FORGE_DTYPE_F16) return launch_i8<fp16_t>(c_dtype, g, p, (int*)work, s);
  return launch_i8<bf16_t>(c_dtype, g, p, (int*)work, s);
}

extern "C" int forge_int8_gemm(const int8_t* a, int64_t lda, const float* row_scale, const int8_t* b, int64_t ldb,
                               const float* col_scale, const void* bias, void* c, int64_t ldc, int c_dtype, int64_t M,
                               int64_t N, int64_t K, void* work, void* stream) {
  return forge_int8_gemm_typed(a, lda, row_scale, b, ldb, col_scale, bias, c_dtype, c, ldc, c_dtype, M, N, K, work, stream);
}

// The rows of x in 8 bits and their product in one call: work holds the integers,
// their scales, and the product's own workspace.
static int64_t rows8_bytes(int64_t M, int64_t kp) { return M * kp + (M * 4 + 15) / 16 * 16; }

extern "C" int64_t forge_int8_linear_workspace(int64_t M, int64_t N, int64_t K) {
  const int64_t own = forge_int8_gemm_workspace(M, N, K);
  return own < 0 ? -1 : rows8_bytes(M, (K + 15) / 16 * 16) + own;
}

extern "C" int forge_int8_linear_typed(int x_dtype, const void* x, int64_t ldx, const float* x_col_scale, const int8_t* w,
                                       int64_t ldw, const float* w_scale, const void* bias, int bias_dtype, void* c, int64_t ldc,
                                       int c_dtype, int64_t M, int64_t N, int64_t K, void* work, void* stream) {
  if (M < 0 || N < 0 || K < 0) return forge_set_error(FORGE_ERR_INVALID, "int8_linear: sizes");
  if (int e = check_types("int8_linear", c_dtype, bias, bias_dtype)) return e;
  if (M == 0 || N == 0) return FORGE_OK;
  if (!work || !aligned16(work)) return forge_set_error(FORGE_ERR_INVALID, "int8_linear: work is NULL or not aligned");
  const int64_t kp = (K + 15) / 16 * 16;
  int8_t* q = (int8_t*)work;
  float* scale = (float*)(q + M * kp);
  // (no columns: every sum is 0, whatever the scales; they are not written)
  if (K > 0)
    if (int e = forge_quantize_rows(x_dtype, x, ldx, x_col_scale, q, kp, scale, M, K, stream)) return e;
  if (K == 0)
    if (int e = forge_zero(scale, M * 4, stream)) return e;
  return forge_int8_gemm_typed(q, kp, scale, w, ldw, w_scale, bias, bias_dtype, c, ldc, c_dtype, M, N, K, q + rows8_bytes(M, kp),
                               stream);
}

extern "C" int forge_int8_linear(int x_dtype, const void* x, int64_t ldx, const float* x_col_scale, const int8_t* w, int64_t ldw,
                                 const float* w_scale, const void* bias, void* c, int64_t ldc, int c_dtype, int64_t M, int64_t N,
                                 int64_t K, void* work, void* stream) {
  return forge_int8_linear_typed(x_dtype, x, ldx, x_col_scale, w, ldw, w_scale, bias, c_dtype, c, ldc, c_dtype, M, N, K, work, stream);
}

// dst[c][r] = src[r][c] of 8-bit values, 64 x 64 tiles through LDS, zeros in the
// columns of dst from `rows` to its pitch.
__global__ __launch_bounds__(256) void transpose_1b_kernel(const int8_t* src, int64_t ld_src, int64_t rows, int64_t cols,
                                                           int8_t* dst, int64_t ld_dst) {
  __shared__ int8_t tile[64][68];
  const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int64_t r = r0 + i / 64, c = c0 + i % 64;
    tile[i / 64][i % 64] = r < rows && c < cols ? src[r * ld_src + c] : (int8_t)0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int64_t c = c0 + i / 64, r = r0 + i % 64;
    if (c < cols && r < ld_dst) dst[c * ld_dst + r] = tile[i % 64][i / 64];
  }
}

extern "C" int forge_transpose_1b(const int8_t* src, int64_t ld_src, int64_t rows, int64_t cols, int8_t* dst,
                                  int64_t ld_dst, void* stream) {
  if (rows < 0 || cols < 0 || ld_src < cols || ld_dst < rows) return forge_set_error(FORGE_ERR_INVALID, "transpose_1b: sizes");
  if (rows == 0 || cols == 0) return FORGE_OK;
  if (!src || !dst) return forge_set_error(FORGE_ERR_INVALID, "transpose_1b: an array is NULL");
  const int64_t x = (ld_dst + 63) / 64, y = (cols + 63) / 64;
  if (x > 0x7fffffff || y > 65535) return forge_set_error(FORGE_ERR_INVALID, "transpose_1b: too large");
  transpose_1b_kernel<<<dim3((unsigned)x, (unsigned)y), 256, 0, (hipStream_t)stream>>>(src, ld_src, rows, cols, dst, ld_dst);
  FORGE_CHECK_LAUNCH();
  return FORGE_OK;
}
