// Log-probabilities of target tokens, and the preference and policy losses
// built on them, forward and backward, for gfx950.
//
// For a row of logits x, a temperature t and a target y:
//     z = x / t,   logp = z_y - log sum_j exp(z_j),
//     dlogp/dx_j = (1{j = y} - exp(z_j - lse)) / t,
// so every loss of the log-probabilities has the gradient c / t (1{j = y} -
// p_j) over a row, with one coefficient c = dloss/dlogp a row.
//
// Passes:
//   lp_partial_kernel   reference and sum of exp over a piece of a row (a long row of
//                       a small batch is split over workgroups);
//   lp_rows_kernel      joins the pieces: logp, and for the policy loss its
//                       value and coefficient;
//   lp_sequences_kernel, lp_pairs_kernel  the preference loss: sums over each
//                       answer, then the pairs;
//   lp_grad_kernel      c / t (1{j = y} - p_j) over every row, zeros where the
//                       target is ignored (those rows are not read).
// Bound by HBM: one read of the kept rows, and for the gradient another and one
// write.  Measured on MI355X, bf16, nothing cached, log-probabilities / gradient:
// 4096 rows of 128256 197 / 342 us (5.3 / 6.1 TB/s; a copy 5.8), 2048 of 50257
// (rows off 16 bytes) 56 / 76, 512 of 32000 14 / 16, 16 of 128256 9 / 5.
//
// Numbers: the softmax runs in base 2, with k = log2(e) / t in two fp32 parts
// (the first alone is a temperature off by up to 2^-24, the same way for every
// token: the sums over a sequence would show it); per row a reference m near the
// max of x and d = sum 2^((x_j - m) k) are fp32, and everything behind them (the
// logarithm, ratios, divergences, sums over a sequence and over the batch) is in
// 64 bits: a sum of thousands of log-probabilities less the reference model's is
// a small difference of large numbers.  p_j is 2^((x_j - m) k) / d.  The rows
// that lp_policy_kernel holds use the first part of k alone and no corrections:
// there a log-probability belongs to its own token's ratio and is not summed.
// Mean error over 4096 16-bit rows of 32000 and 128256 at t = 1 and 0.7, with and
// without masked columns: up to 1.2e-8 from lp_partial_kernel, 4e-8 to 6e-8 held
// (rms 1.3e-7 and 1.5e-7, most of it the rounding of the result to fp32).  (One fma
// x_j k - m k would do where m is moderate, but its result at x_j = m is the
// rounding error of m k, which is no longer small where every logit of a row is
// a mask's -1e30.)  A row with a NaN or +infinity, or with nothing but
// -infinity, comes out as NaN; so does a row whose target is outside [0, V)
// without being ignored, of which nothing is read.
#include <initializer_list>
#include <type_traits>

#include "common.h"

namespace {

constexpr int kBlock = 256;
constexpr int kWave = 64;
constexpr int kU = 4;                   // vectors in flight per thread (2: the same; 8: 5% slower, 20% at 512 rows of 32000)
constexpr int kMaxSplits = 64;          // pieces of a row
constexpr int64_t kMaxGrid = 1 << 22;   // workgroups of a launch; more work loops
constexpr double kLn2 = 0.693147180559945309417;

struct Rows {
  const void* x; int64_t xn, xs;          // logits [N, S, V]: element strides of N and S
  const int64_t* target; int64_t tn, ts;
  int64_t n, s, v;                        // N, S, V
  int64_t ignore;
  float k, k_lo;                          // log2(e) / temperature, and what its rounding to fp32 leaves
};

// What the passes hand on.
struct Work {
  float2* part;   // [N * S][splits]: (reference, sum) of each piece
  int splits;
  float2* state;  // [N * S]: (m, 1 / d)
  float* logps;   // [N, S]
  double* row64;  // [N * S]: policy: weighted loss
  float* coef;    // policy [N * S]
  int* counts;    // [N] kept tokens of each sequence, then tokens and sequences that have any
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^(far k): the exponent p = far k is rounded; what that and k_lo leave is
// added to first order as rest += 2^p (far k - p + far k_lo).  Where 2^p is not
// 0 that difference is below 2^-16; where p is infinite it is infinite or NaN,
// and held between -1 and 1 (a NaN gives -1) 2^p = 0 times it is 0, so that
// masked columns leave the others' rest as it is.
__device__ __forceinline__ float exp2_rest(float far, float k, float k_lo, float& rest) {
  const float p = far * k, e = fast_exp2(p);
  rest = fmaf(e, __builtin_amdgcn_fmed3f(fmaf(far, k_lo, fmaf(far, k, -p)), -1.f, 1.f), rest);
  return e;
}

__device__ __forceinline__ float with_rest(float sum, float rest) { return fmaf(rest, (float)kLn2, sum); }

// Sum of 2^((v - at) k) over N values, which are overwritten.  16-bit logits
// take few values near the maximum, and most rows of a batch have much the same
// maximum, so the rounding errors of the exponents, and of adding those few
// exponentials to a long sum, are the same in row after row, and the sum over an
// answer adds them up: hence the rest, and a sum in pairs.  Mean error of a
// log-probability over bf16 rows of 128256: 1e-7 with neither, 3e-9 with both.
template <int N>
__device__ __forceinline__ float sum_exp2(float (&v)[N], float at, const Rows& a) {
  float rest = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = exp2_rest(v[j] - at, a.k, a.k_lo, rest);
#pragma unroll
  for (int w = 1; w < N; w *= 2)
#pragma unroll
    for (int j = 0; j + w < N; j += 2 * w) v[j] += v[j + w];
  return with_rest(v[0], rest);
}

// The factor that takes a sum of 2^((x - m) k) to the reference `to` >= m; 0 for
// an empty sum (m = -inf).  One factor a thread and one a piece: each factor's
// error is that of a few values again, and a chain of them (a tree of pairs,
// each to its larger reference) left another 2.5e-8.
__device__ __forceinline__ float factor_to(float m, float to, const Rows& a) {
  const float far = m - (to == -INFINITY ? 0.f : to);
  float rest = 0.f;
  const float e = exp2_rest(far, a.k, a.k_lo, rest);
  return with_rest(e, rest);
}

// 16 bytes at an address that is a multiple of the element only (global memory
// takes them at any).
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <class T, bool NT>
__device__ __forceinline__ Vec16<T> load_any(const T* p) {
  const u32x4_any* q = reinterpret_cast<const u32x4_any*>(p);
  const u32x4_any w = NT ? __builtin_nontemporal_load(q) : *q;
  Vec16<T> t;
  t.raw = make_uint4(w.x, w.y, w.z, w.w);
  return t;
}

template <class T>
__device__ __forceinline__ void store_any(T* p, const Vec16<T>& t) {
  const u32x4_any w = {t.raw.x, t.raw.y, t.raw.z, t.raw.w};
  __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any*>(p));
}

__device__ __forceinline__ int64_t target_of(const Rows& a, int64_t row) {
  const int64_t n = row / a.s, s = row - n * a.s;
  return a.target[n * a.tn + s * a.ts];
}

template <class T>
__device__ __forceinline__ const T* row_of(const Rows& a, int64_t row) {
  const int64_t n = row / a.s, s = row - n * a.s;
  return (const T*)a.x + (n * a.xn + s * a.xs);
}

__device__ __forceinline__ bool in_vocab(const Rows& a, int64_t y) { return y >= 0 && y < a.v; }

// Sum over the workgroup in a fixed order; every thread gets it.
template <class V, int NT>
__device__ __forceinline__ V block_total(V v, V* red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  V t = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) t += red[i];
  return t;
}

// The largest over the workgroup (a NaN does not count); every thread gets it.
template <int NT>
__device__ __forceinline__ float block_largest(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) t = fmaxf(t, red[i]);
  return t;
}

// counts[n]: tokens of sequence n that are not ignored; counts[N], counts[N + 1]:
// tokens in all and sequences that have any.  By one workgroup: a wave to a
// sequence, or several where there are fewer sequences than waves (a packed batch
// is one long sequence).
template <int NT>
__device__ void count_tokens(const Rows& a, int* counts) {
  constexpr int NW = NT / 64;
  __shared__ int red[NW], part[NW];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  auto count = [&](int64_t n, int first, int step) {  // by a wave: tokens first * 64 + lane, + step * 64, ...
    int c = 0;
#pragma unroll 8
    for (int64_t s = first * 64 + lane; s < a.s; s += step * 64) c += a.target[n * a.tn + s * a.ts] != a.ignore;
    for (int off = 32; off >= 1; off >>= 1) c += __shfl_xor(c, off, 64);
    return c;
  };
  int tokens = 0, filled = 0;
  auto store = [&](int64_t n, int c) {
    counts[n] = c;
    tokens += c;
    filled += c > 0;
  };
  if (a.n >= NW) {
    for (int64_t n = wave; n < a.n; n += NW) {
      const int c = count(n, 0, 1);
      if (lane == 0) store(n, c);
    }
  } else {
    const int each = NW / (int)a.n;  // waves of a sequence
    const int n = wave / each;
    const int c = n < a.n ? count(n, wave % each, each) : 0;
    if (lane == 0) part[wave] = c;
    __syncthreads();
    if ((int)threadIdx.x < a.n) {
      int t = 0;
      for (int w = 0; w < each; ++w) t += part[threadIdx.x * each + w];
      store(threadIdx.x, t);
    }
  }
  tokens = block_total<int, NT>(tokens, red);
  filled = block_total<int, NT>(filled, red);
  if (threadIdx.x == 0) {
    counts[a.n] = tokens;
    counts[a.n + 1] = filled;
  }
}

// ---------------------------------------------------------------------------
// reference and sum of a piece of a row
// ---------------------------------------------------------------------------
template <class T, int NT>
__global__ __launch_bounds__(NT) void lp_partial_kernel(Rows a, Work w, bool count) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ float red[NT / 64];
  const int tid = threadIdx.x;
  int64_t first = blockIdx.x, step = gridDim.x;
  if (count) {  // workgroup 0 counts
    if (blockIdx.x == 0) {
      count_tokens<NT>(a, w.counts);
      return;
    }
    first -= 1;
    step -= 1;
  }
  const int64_t pieces = a.n * a.s * w.splits;
  for (int64_t i = first; i < pieces; i += step) {
    const int64_t row = i / w.splits;
    const int piece = (int)(i - row * w.splits);
    const int64_t y = target_of(a, row);
    if (y == a.ignore || !in_vocab(a, y)) continue;  // (uniform over the workgroup)
    const T* x = row_of<T>(a, row);
    const int64_t nvec = a.v / VEC, per = (nvec + w.splits - 1) / w.splits;
    const int64_t lo = piece * per, hi = lo + per < nvec ? lo + per : nvec;
    // m is a reference that no value so far exceeds by more than the headroom
    // (2^40 in a sum), so that it hardly ever moves
    const float headroom = 40.f / a.k;
    float m = -INFINITY, d = 0.f;
    auto take = [&](auto& v) {
      constexpr int N = sizeof(v) / sizeof(float);
      float t = v[0];
#pragma unroll
      for (int j = 1; j < N; ++j) t = fmaxf(t, v[j]);
      if (t > m + headroom) {
        d *= factor_to(m, t, a);
        m = t;
      }
      d += sum_exp2(v, m == -INFINITY ? 0.f : m, a);
    };
    int64_t c = lo;
    for (; c + NT * kU <= hi; c += NT * kU) {
      Vec16<T> t[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) t[u] = load_any<T, false>(x + (c + u * NT + tid) * VEC);
      float v[kU * VEC];
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[u * VEC + j] = to_f32(t[u].v[j]);
      take(v);
    }
    for (c += tid; c < hi; c += NT) {
      const Vec16<T> t = load_any<T, false>(x + c * VEC);
      float v[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = to_f32(t.v[j]);
      take(v);
    }
    if (piece == w.splits - 1 && nvec * VEC + tid < a.v) {  // the columns behind the last vector
      float v[1] = {to_f32(x[nvec * VEC + tid])};
      take(v);
    }
    const float to = block_largest<NT>(m, red);
    d = block_total<float, NT>(d * factor_to(m, to, a), red);
    if (tid == 0) w.part[i] = make_float2(to, d);
  }
}

// ---------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------
// log-probability in 64 bits from a row's m, d and its target's logit.
__device__ __forceinline__ double logp_of(const Rows& a, float xy, float m, float d) {
  return kLn2 * (((double)xy - (double)m) * ((double)a.k + (double)a.k_lo) - log2((double)d));
}

// The row's pieces joined over `lanes` neighbouring lanes (a power of two, at
// least the splits); lane 0 of them returns the log-probability and stores the
// row's state.  An ignored row gives 0, a target out of range NaN.
template <class T>
__device__ __forceinline__ double join_row(const Rows& a, const Work& w, int64_t row, int lane, int lanes, int64_t y) {
  const bool kept = y != a.ignore && in_vocab(a, y);
  float m = -INFINITY, d = 0.f;
  if (kept && lane < w.splits) {
    const float2 p = w.part[row * w.splits + lane];
    m = p.x;
    d = p.y;
  }
  if (lanes > 1) {
    float to = m;
    for (int off = lanes >> 1; off >= 1; off >>= 1) to = fmaxf(to, __shfl_xor(to, off, 64));
    d *= factor_to(m, to, a);
    for (int off = lanes >> 1; off >= 1; off >>= 1) d += __shfl_xor(d, off, 64);
    m = to;
  }
  if (lane != 0) return 0.0;
  double lp = y == a.ignore ? 0.0 : __builtin_nan("");
  if (kept) lp = logp_of(a, to_f32(row_of<T>(a, row)[y]), m, d);
  if (w.state) w.state[row] = make_float2(m, 1.f / d);
  w.logps[row] = (float)lp;
  return lp;
}

struct Policy {
  const float* adv; int64_t an, as;
  const float* old; int64_t on, os;  // nullptr: the policy itself (ratio 1)
  const float* ref; int64_t rn, rs;  // nullptr: no divergence
  double low, high, beta;            // clip range, weight of the divergence
  int reduction;
  float* kl;                         // [N, S]
  const float* scale;                // of the gradient, or nullptr (1)
};

// A token's loss -min(r A, clip(r) A) + beta (e^f - f - 1), with r = exp(logp -
// old) and f = ref - logp, and its derivative by logp.
__device__ __forceinline__ void policy_token(const Policy& p, int64_t n, int64_t s, double lp, double& loss, double& d,
                                             float& kl) {
  const double adv = p.adv[n * p.an + s * p.as];
  const double r = p.old ? exp(lp - (double)p.old[n * p.on + s * p.os]) : lp == lp ? 1.0 : lp;
  const double clipped = r < p.low ? p.low : r > p.high ? p.high : r;
  const double u = r * adv, c = clipped * adv;
  const bool moves = !(u > c);  // the unclipped term is the smaller one, or NaN
  loss = moves ? -u : -c;
  d = moves ? -u : 0.0;
  kl = 0.f;
  if (p.ref) {
    const double f = (double)p.ref[n * p.rn + s * p.rs] - lp, e = expm1(f);
    const double far = f == INFINITY ? f : e - f;
    kl = (float)far;
    if (p.beta != 0.0) {  // (where it is only reported an infinite one may not reach the loss: 0 times it is NaN)
      loss += p.beta * far;
      d -= p.beta * e;
    }
  }
}

// Weight of a kept token of sequence n in the loss.
__device__ __forceinline__ double token_weight(const Rows& a, const int* counts, int reduction, int64_t n) {
  if (reduction == FORGE_REDUCE_MEAN) return 1.0 / (double)counts[a.n];
  if (reduction == FORGE_REDUCE_SEQUENCE) return 1.0 / ((double)counts[a.n + 1] * (double)counts[n]);
  return 1.0;
}

template <class T, bool POLICY>
__global__ __launch_bounds__(kBlock) void lp_rows_kernel(Rows a, Work w, Policy p, int lanes) {
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t rows = a.n * a.s, step = (int64_t)gridDim.x * (kBlock / lanes);
  for (int64_t row = (int64_t)blockIdx.x * (kBlock / lanes) + threadIdx.x / lanes; row < rows; row += step) {
    const int64_t n = row / a.s, s = row - n * a.s;
    const int64_t y = a.target[n * a.tn + s * a.ts];
    const double lp = join_row<T>(a, w, row, lane, lanes, y);
    if constexpr (POLICY) {
      if (lane == 0) {
        double loss = 0.0, d = 0.0;
        float kl = 0.f;
        if (y != a.ignore) {
          policy_token(p, n, s, lp, loss, d, kl);
          const double weight = token_weight(a, w.counts, p.reduction, n);
          loss *= weight;
          d *= weight;
          if (p.scale) d *= (double)*p.scale;
        }
        w.row64[row] = loss;
        w.coef[row] = (float)d;
        p.kl[row] = kl;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// preference loss
// ---------------------------------------------------------------------------
// seq[n] = sum (or mean) of sequence n's log-probabilities, in a fixed order; a
// workgroup to a sequence.
template <class T>
__global__ __launch_bounds__(1024) void lp_sequences_kernel(Rows a, Work w, int lanes, bool mean, double* seq) {
  __shared__ double redd[16];
  __shared__ int redi[16];
  const int lane = threadIdx.x & (lanes - 1), per = 1024 / lanes;
  for (int64_t n = blockIdx.x; n < a.n; n += gridDim.x) {
    double sum = 0.0;
    int count = 0;
    for (int64_t s = threadIdx.x / lanes; s < a.s; s += per) {
      const int64_t y = a.target[n * a.tn + s * a.ts];
      const double lp = join_row<T>(a, w, n * a.s + s, lane, lanes, y);
      if (lane == 0) {
        sum += lp;
        count += y != a.ignore;
      }
    }
    sum = block_total<double, 1024>(sum, redd);
    count = block_total<int, 1024>(count, redi);
    if (threadIdx.x == 0) {
      seq[n] = mean && count ? sum / count : sum;
      w.counts[n] = count;
    }
  }
}

struct Pairs {
  const double* seq;   // [2 P]: chosen answers, then rejected ones
  const int* counts;
  const float* ref;    // [2 P] or nullptr
  int64_t pairs;
  double beta, smoothing;
  int kind, reduction;
  bool mean;           // seq holds means
  float* loss;         // one value, or [P] with FORGE_REDUCE_NONE
  float* logps;        // [2 P]
  float* rewards;      // [2 P]
  float* coef;         // [2 P]: dloss / dlogp of each token of a sequence
};

// h = beta ((chosen - its reference) - (rejected - its reference)):
//   sigmoid  -(1 - e) log s(h) - e log s(-h), slope beta (e - s(-h)) with
//            e the label smoothing
//   hinge    max(0, 1 - h)
//   ipo      (h / beta - 1 / (2 beta))^2
__global__ __launch_bounds__(kBlock) void lp_pairs_kernel(Pairs p) {
  __shared__ double red[kBlock / 64];
  double total = 0.0;
  for (int64_t i = threadIdx.x; i < p.pairs; i += kBlock) {
    const int64_t j = i + p.pairs;
    const double over = p.seq[i] - (p.ref ? (double)p.ref[i] : 0.0), under = p.seq[j] - (p.ref ? (double)p.ref[j] : 0.0);
    const double h = p.beta * (over - under);
    double loss, d;  // d = dloss / d(over)
    if (p.kind == FORGE_PREF_SIGMOID) {
      const double tail = log1p(exp(-fabs(h)));
      const double up = tail + (h < 0.0 ? -h : 0.0), down = tail + (h > 0.0 ? h : 0.0);  // -log s(h), -log s(-h)
      // (a term of weight 0 may be infinite)
      loss = (p.smoothing < 1.0 ? (1.0 - p.smoothing) * up : 0.0) + (p.smoothing > 0.0 ? p.smoothing * down : 0.0);
      d = p.beta * (p.smoothing - 1.0 / (1.0 + exp(h)));
    } else if (p.kind == FORGE_PREF_HINGE) {
      loss = h >= 1.0 ? 0.0 : 1.0 - h;  // (a NaN stays)
      d = h >= 1.0 ? 0.0 : h == h ? -p.beta : h;
    } else {
      const double t = over - under - 0.5 / p.beta;
      loss = t * t;
      d = 2.0 * t;
    }
    const double weight = p.reduction == FORGE_REDUCE_MEAN ? 1.0 / (double)p.pairs : 1.0;
    if (p.reduction == FORGE_REDUCE_NONE) p.loss[i] = (float)loss;
    total += weight * loss;
    d *= weight;
    p.logps[i] = (float)p.seq[i];
    p.logps[j] = (float)p.seq[j];
    p.rewards[i] = (float)(p.beta * over);
    p.rewards[j] = (float)(p.beta * under);
    p.coef[i] = (float)(p.mean && p.counts[i] ? d / p.counts[i] : d);
    p.coef[j] = (float)(-(p.mean && p.counts[j] ? d / p.counts[j] : d));
  }
  total = block_total<double, kBlock>(total, red);
  if (threadIdx.x == 0 && p.reduction != FORGE_REDUCE_NONE) p.loss[0] = (float)total;
}

// ---------------------------------------------------------------------------
// gradient
// ---------------------------------------------------------------------------
struct Grad {
  void* out; int64_t on, os;              // [N, S, V]; may be the logits themselves
  const float* coef; int64_t cn, cs;      // dloss/dlogp of token (n, s)
  const float* up; int64_t us, un;        // times up[(n % un) * us] where given
  const float2* state;
  const float* logps;
  float inv_t;                            // 1 / temperature
  const double* rows64;                   // workgroup 0 sums these ...
  float* sum;                             // ... into here, where given
};

// Vectors of a thread: 4096 rows of 128256, 342 us; with 1 576, 2 378, 8 348 (8
// on 2048 rows of 50257: 95 against 76).
constexpr int kGradVec = 4;

// *sum = the rows' losses in a fixed order, by one workgroup.
template <int NT>
__device__ void sum_rows(const double* rows, int64_t n, float* sum, double* red) {
  double t = 0.0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < n; i += NT) t += rows[i];
  t = block_total<double, NT>(t, red);
  if (threadIdx.x == 0) *sum = (float)t;
}

template <class T, int NT>
__global__ __launch_bounds__(NT) void lp_grad_kernel(Rows a, Grad g, int64_t chunks) {
  constexpr int VEC = 16 / sizeof(T);
  const int tid = threadIdx.x;
  int64_t first = blockIdx.x, step = gridDim.x;
  if (g.sum) {
    if (blockIdx.x == 0) {
      __shared__ double red[NT / 64];
      sum_rows<NT>(g.rows64, a.n * a.s, g.sum, red);
      return;
    }
    first -= 1;
    step -= 1;
  }
  const int64_t items = a.n * a.s * chunks;
  for (int64_t i = first; i < items; i += step) {
    const int64_t row = i / chunks, chunk = i - row * chunks;
    const int64_t n = row / a.s, s = row - n * a.s;
    const int64_t y = a.target[n * a.tn + s * a.ts];
    const T* x = (const T*)a.x + (n * a.xn + s * a.xs);
    T* o = (T*)g.out + (n * g.on + s * g.os);
    float c = 0.f;
    if (y != a.ignore) {
      c = g.coef[n * g.cn + s * g.cs] * g.inv_t;
      if (g.up) c *= g.up[(n % g.un) * g.us];
      if (!in_vocab(a, y)) c = __builtin_nanf("");
    }
    const int64_t nvec = a.v / VEC;
    const int64_t c0 = chunk * (NT * kGradVec);
    const bool last = chunk == chunks - 1;
    if (c == 0.f) {  // nothing to read
      Vec16<T> z;
      z.raw = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int u = 0; u < kGradVec; ++u)
        if (const int64_t at = c0 + u * NT + tid; at < nvec) store_any(o + at * VEC, z);
      if (last && nvec * VEC + tid < a.v) o[nvec * VEC + tid] = from_f32<T>(0.f);
      continue;
    }
    const float2 st = g.state[row];
    const float scale = -c * st.y, m = st.x;
    const float at_y = -c * expm1f(g.logps[row]);  // c (1 - p), without its cancellation near 1
    Vec16<T> t[kGradVec];
#pragma unroll
    for (int u = 0; u < kGradVec; ++u)
      if (const int64_t at = c0 + u * NT + tid; at < nvec) t[u] = load_any<T, true>(x + at * VEC);
#pragma unroll
    for (int u = 0; u < kGradVec; ++u) {
      const int64_t at = c0 + u * NT + tid;
      if (at >= nvec) continue;
      const int64_t hit = y - at * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float v = scale * fast_exp2((to_f32(t[u].v[j]) - m) * a.k);
        if (hit == j) v = at_y;
        t[u].v[j] = from_f32<T>(v);
      }
      store_any(o + at * VEC, t[u]);
    }
    if (last && nvec * VEC + tid < a.v) {
      const int64_t at = nvec * VEC + tid;
      const float v = scale * fast_exp2((to_f32(x[at]) - m) * a.k);
      o[at] = from_f32<T>(at == y ? at_y : v);
    }
  }
}

// ---------------------------------------------------------------------------
// policy loss with a row held on chip
//
// One workgroup a row of 16-bit logits (512 threads; a wave where many rows are
// short), which is read once and written once: thread t of NT owns the 16-byte
// vectors t + NT i, the first NL in LDS
// (filled by loads that go there by themselves), the others in registers (8 + 24
// vectors: 131072 columns, two workgroups on a CU; one computes while the other
// loads or stores).
//   A  the largest value, as packed 16-bit integers (bits of non-negative values
//      are in their order; a row of negative ones takes a second look)
//   B  d = sum of 2^(x k - m k)
//   C  one thread, in 64 bits: the token's loss and coefficient
//   D  the gradient, each exponential again (kept in 16 bits it would be rounded
//      twice)
// Measured on MI355X, bf16 [8, 1024, 128256], 66% of the rows kept, nothing
// cached, least of 24: 654 us, 5.3 TB/s of reads and writes (a copy 5.8), against
// 818 us for the passes above, which read those rows twice at 5.9 TB/s (on
// average 663 and 857).
// One fma gives x k - m k: what rounding m k leaves is the same factor on every
// exponential and on d, and the log-probability takes it into account.  Where m k
// passes 2^29 (a row of a mask's lowest values) that factor could leave fp32;
// values that differ are then 2^17 apart or more in the exponent, so a power of
// two in place of k, whose products are exact, gives the same 1 or 0.  1 does
// where that product leaves fp32 (bf16 near its largest, t up to 0.72): k is
// below 2^21, so |m| is 2^107 or more and values that differ are 2^98 apart.
// ---------------------------------------------------------------------------
constexpr int kRow = 512;  // threads of a row

typedef short short2_t __attribute__((ext_vector_type(2)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const void* base, uint32_t bytes) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)b);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), (short)0, (int)bytes,
                                           0x00020000);
}

template <class T, int NT, int NL, int NR>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(NR > 8 ? 4 : 6))) void lp_policy_kernel(
    Rows a, Work w, Policy p, Grad g) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ __attribute__((aligned(16))) uint4 lds[NL > 0 ? NL * NT : 1];
  __shared__ float red[NT / 64], say[2];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x, n = row / a.s, s = row - n * a.s;
  const int64_t y = a.target[n * a.tn + s * a.ts];
  const T* x = (const T*)a.x + (n * a.xn + s * a.xs);
  T* o = (T*)g.out + (n * g.on + s * g.os);
  const int nvec = (int)(a.v / VEC), tail = (int)(a.v - (int64_t)nvec * VEC);
  auto on = [&](int i) { return tid < nvec - i * NT; };
  auto fill = [&](float f) {
    Vec16<T> z;
#pragma unroll
    for (int j = 0; j < VEC; ++j) z.v[j] = from_f32<T>(f);
    for (int i = tid; i < nvec; i += NT) store_any(o + (int64_t)i * VEC, z);
    if (tid < tail) o[(int64_t)nvec * VEC + tid] = from_f32<T>(f);
  };
  if (y == a.ignore || !in_vocab(a, y)) {
    const float f = y == a.ignore ? 0.f : __builtin_nanf("");
    if (tid == 0) {
      w.logps[row] = f;
      w.row64[row] = f;
      p.kl[row] = p.ref ? f : 0.f;
    }
    fill(f);
    return;
  }

  uint4 reg[NR];
  if constexpr (NL > 0) {
    const __amdgpu_buffer_rsrc_t rs = row_rsrc(x, (uint32_t)(nvec * 16));
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (on(i)) {
        __attribute__((address_space(3))) char* dst =
            (__attribute__((address_space(3))) char*)lds + (i * (NT / 64) + wave) * 1024;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, (uint32_t)tid * 16u,
                                                 i * NT * 16, 0, 2);
      }
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    reg[i] = make_uint4(0, 0, 0, 0);
    if (on(NL + i)) reg[i] = load_any<T, true>(x + ((int64_t)(NL + i) * NT + tid) * VEC).raw;
  }
  const float last = tid < tail ? to_f32(x[(int64_t)nvec * VEC + tid]) : -INFINITY;
  const float xy = to_f32(x[y]);
  if constexpr (NL > 0) {
    __builtin_amdgcn_s_waitcnt(0);  // this wave's part of lds is there
    __syncthreads();                // and every other's
  }
  uint4* mine = lds + tid;
  auto each = [&](auto f) {  // f(vector, its index)
#pragma unroll 1
    for (int i = 0; i < NL; ++i)
      if (on(i)) f(mine[i * NT], i);
#pragma unroll
    for (int i = 0; i < NR; ++i)
      if (on(NL + i)) f(reg[i], NL + i);
  };
  auto unpack = [](const uint4& r, float (&v)[VEC]) {
    Vec16<T> t;
    t.raw = r;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = to_f32(t.v[j]);
  };

  // A
  short2_t mi = {(short)0x8000, (short)0x8000};
  each([&](const uint4& r, int) {
    mi = __builtin_elementwise_max(mi, __builtin_bit_cast(short2_t, r.x));
    mi = __builtin_elementwise_max(mi, __builtin_bit_cast(short2_t, r.y));
    mi = __builtin_elementwise_max(mi, __builtin_bit_cast(short2_t, r.z));
    mi = __builtin_elementwise_max(mi, __builtin_bit_cast(short2_t, r.w));
  });
  const short top = mi.x > mi.y ? mi.x : mi.y;
  float m = top >= 0 ? to_f32(__builtin_bit_cast(T, top)) : -INFINITY;
  m = block_largest<NT>(fmaxf(m, last), red);
  if (m < 0.f) {  // nothing that is not negative but perhaps in the tail
    each([&](const uint4& r, int) {
      float v[VEC];
      unpack(r, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) m = fmaxf(m, v[j]);
    });
    m = block_largest<NT>(m, red);
  }
  float k = a.k, mk = m * k;
  const bool far = fabsf(mk) >= 0x1p29f && fabsf(m) < INFINITY;
  if (far) {
    k = __uint_as_float(__float_as_uint(k) & 0x7f800000);
    if (!(fabsf(m * k) < INFINITY)) k = 1.f;
    mk = m * k;
  }

  // B
  float d = fast_exp2(fmaf(last, k, -mk));  // (0 without a tail)
  each([&](const uint4& r, int) {
    float v[VEC];
    unpack(r, v);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = fast_exp2(fmaf(v[j], k, -mk));
#pragma unroll
    for (int h = VEC / 2; h >= 1; h /= 2)
#pragma unroll
      for (int j = 0; j < h; ++j) v[j] += v[j + h];
    d += v[0];
  });
  d = block_total<float, NT>(d, red);

  // C
  if (tid == 0) {
    const double z = far ? ((double)xy - (double)m) * (double)a.k : (double)xy * (double)k - (double)mk;
    const double lp = kLn2 * (z - log2((double)d));
    double loss, dl;
    float kl;
    policy_token(p, n, s, lp, loss, dl, kl);
    const double weight = token_weight(a, w.counts, p.reduction, n);
    w.logps[row] = (float)lp;
    w.row64[row] = loss * weight;
    p.kl[row] = kl;
    const float c = (float)(p.scale ? dl * weight * (double)*p.scale : dl * weight) * g.inv_t;
    say[0] = c == 0.f ? 0.f : -c / d;
    say[1] = c == 0.f ? 0.f : -c * (float)expm1(lp);
  }
  __syncthreads();
  const float scale = say[0], at_y = say[1];

  // D
  if (scale == 0.f && at_y == 0.f) {
    fill(0.f);
    return;
  }
  each([&](const uint4& r, int i) {
    float v[VEC];
    unpack(r, v);
    Vec16<T> t;
#pragma unroll
    for (int j = 0; j < VEC; ++j) t.v[j] = from_f32<T>(scale * fast_exp2(fmaf(v[j], k, -mk)));
    store_any(o + ((int64_t)i * NT + tid) * VEC, t);
  });
  if (tid < tail) o[(int64_t)nvec * VEC + tid] = from_f32<T>(scale * fast_exp2(fmaf(last, k, -mk)));
  // the target's column by the thread that has stored it, after that store
  const int64_t yv = y / VEC;
  if (yv < nvec ? (int)(yv % NT) == tid : (int)(y - (int64_t)nvec * VEC) == tid) o[y] = from_f32<T>(at_y);
}

__global__ __launch_bounds__(1024) void lp_count_kernel(Rows a, int* counts) { count_tokens<1024>(a, counts); }

__global__ __launch_bounds__(1024) void lp_sum_kernel(const double* rows, int64_t n, float* sum) {
  __shared__ double red[16];
  sum_rows<1024>(rows, n, sum, red);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int vec_of(int dtype) { return (int)(16 / dtype_size(dtype)); }

// Pieces of a row: enough workgroups for the card (4 on each CU), none with
// less than a vector a thread.  512 rows of 32000 / 16 of 128256: 13.7 / 9.0 us;
// with 2 on each CU 14.0 / 8.0, 8 14.9 / 9.0, 16 17.5 / 8.9.  (Rows that a wave
// takes: 512 to 1023 of them in two pieces from 512 vectors on, else in one.)
int splits_for(int64_t rows, int64_t v, int dtype) {
  const int64_t most = v / ((int64_t)vec_of(dtype) * kBlock);
  int64_t s = rows ? (1024 + rows - 1) / rows : 1;
  if (s > most) s = most;
  if (s > kMaxSplits) s = kMaxSplits;
  return s < 1 ? 1 : (int)s;
}

int lanes_of(int splits) {
  int l = 1;
  while (l < splits) l <<= 1;
  return l;
}

int64_t align16(int64_t b) { return (b + 15) / 16 * 16; }

// One call's workspace: the pieces, the rows' losses and coefficients, counts.
struct Layout {
  int64_t part, row64, coef, counts, seq, state, bytes;
  int splits;
  Layout(int dtype, int64_t n, int64_t s, int64_t v) {
    const int64_t rows = n * s;
    splits = splits_for(rows, v, dtype);
    part = 0;
    row64 = align16(part + rows * splits * (int64_t)sizeof(float2));
    coef = align16(row64 + rows * (int64_t)sizeof(double));
    counts = align16(coef + rows * (int64_t)sizeof(float));
    seq = align16(counts + (n + 2) * (int64_t)sizeof(int));
    state = align16(seq + n * (int64_t)sizeof(double));
    bytes = state + rows * (int64_t)sizeof(float2);
  }
  Work work(void* base, float* logps, float2* state_out) const {
    char* b = (char*)base;
    Work w;
    w.part = (float2*)(b + part);
    w.splits = splits;
    w.state = state_out;
    w.logps = logps;
    w.row64 = (double*)(b + row64);
    w.coef = (float*)(b + coef);
    w.counts = (int*)(b + counts);
    return w;
  }
};

// Many rows of few vectors take a workgroup of one wave each.  Measured on
// MI355X, bf16, log-probabilities / gradient / policy loss with 256 (512) threads
// and with 64: 32768 (policy 16384) rows of 1003 77 / 73 / 87 us and 33 / 37 / 33;
// of 4096 95 / 101 / 99 and 58 / 88 / 56; 16384 of 8192 68 / 89 / 118 and 56 / 86
// / 106.  64 rows of 4000: 6.4 / 4.1 and 7.3 / 4.8.
constexpr int kSmallVecs = 1024, kSmallRows = 512;

bool small_rows(int dtype, const Rows& a) {
  return a.v / vec_of(dtype) <= kSmallVecs && a.n * a.s >= kSmallRows;
}

unsigned capped(int64_t blocks) { return (unsigned)(blocks > kMaxGrid ? kMaxGrid : blocks); }

int check_rows(const char* what, int dtype, const Rows& a, double temperature) {
  if (a.n < 0 || a.s < 0 || a.v < 0) return forge_set_error(FORGE_ERR_INVALID, "%s: negative shape", what);
  if (dtype != FORGE_DTYPE_F32 && dtype != FORGE_DTYPE_BF16 && dtype != FORGE_DTYPE_F16)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  if (!(temperature >= 1e-6 && temperature <= 1e6))
    return forge_set_error(FORGE_ERR_INVALID, "%s: temperature %g (1e-6 to 1e6)", what, temperature);
  const int64_t lim = 0x7fffffff;
  if (a.n > lim || a.s > lim || a.v > lim || a.n * a.s > lim)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: 2^31 rows or columns", what);
  if (a.n * a.s > 0 && a.v == 0) return forge_set_error(FORGE_ERR_INVALID, "%s: no columns", what);
  return FORGE_OK;
}

// The arrays that a call with rows cannot do without.
int check_given(const char* what, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (!p) return forge_set_error(FORGE_ERR_INVALID, "%s: a required pointer is NULL", what);
  return FORGE_OK;
}

template <class F>
int by_dtype(int dtype, F f) {
  if (dtype == FORGE_DTYPE_F32) f((float*)nullptr);
  else if (dtype == FORGE_DTYPE_BF16) f((bf16_t*)nullptr);
  else f((fp16_t*)nullptr);
  FORGE_CHECK_LAUNCH();
  return FORGE_OK;
}

int launch_partial(int dtype, const Rows& a, const Work& w, bool count, hipStream_t s) {
  const unsigned grid = capped(a.n * a.s * w.splits) + (count ? 1u : 0u);
  return by_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (small_rows(dtype, a)) lp_partial_kernel<T, kWave><<<grid, kWave, 0, s>>>(a, w, count);
    else lp_partial_kernel<T, kBlock><<<grid, kBlock, 0, s>>>(a, w, count);
  });
}

int launch_rows(int dtype, const Rows& a, const Work& w, const Policy* p, hipStream_t s) {
  const int lanes = lanes_of(w.splits), per = kBlock / lanes;
  const unsigned grid = capped((a.n * a.s + per - 1) / per);
  return by_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (p) lp_rows_kernel<T, true><<<grid, kBlock, 0, s>>>(a, w, *p, lanes);
    else lp_rows_kernel<T, false><<<grid, kBlock, 0, s>>>(a, w, Policy{}, lanes);
  });
}

int launch_grad(int dtype, const Rows& a, const Grad& g, bool rows, hipStream_t s) {
  const bool small = small_rows(dtype, a);
  const int64_t per = (int64_t)vec_of(dtype) * (small ? kWave : kBlock) * kGradVec;
  const int64_t chunks = (a.v + per - 1) / per;
  const unsigned grid = (rows ? capped(a.n * a.s * chunks) : 0u) + (g.sum ? 1u : 0u);
  return by_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (small) lp_grad_kernel<T, kWave><<<grid, kWave, 0, s>>>(a, g, chunks);
    else lp_grad_kernel<T, kBlock><<<grid, kBlock, 0, s>>>(a, g, chunks);
  });
}

// The kernel that holds a row, where it takes this call: 16-bit logits whose row
// fits (in registers alone at any alignment), and a row for every CU.  Measured
// on MI355X, bf16, 128256 columns, against rows split over workgroups and read
// twice: 64 rows 26 / 22 us, 128 28 / 29, 256 36 / 43, 512 49 / 73, 2048 202 /
// 258; 32000 columns, 512 rows 23 / 30, 2048 57 / 75; 50257 (rows off 16 bytes),
// 2048 rows 96 / 122.
constexpr int64_t kResidentRows = 256;

template <class T>
bool launch_policy(const Rows& a, const Work& w, const Policy& p, const Grad& g, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    const int64_t rows = a.n * a.s, nvec = a.v / 8, per = (nvec + kRow - 1) / kRow;  // vectors of a thread
    if (rows < kResidentRows || rows > kMaxGrid || per > 32) return false;
    const bool aligned = aligned16(a.x) && a.xn % 8 == 0 && a.xs % 8 == 0;
    if (per > 16 && !aligned) return false;
    const unsigned grid = (unsigned)rows;
    lp_count_kernel<<<1, 1024, 0, s>>>(a, w.counts);
    const bool small = nvec <= kSmallVecs && rows >= kSmallRows;
    if (small && nvec <= 8 * kWave) lp_policy_kernel<T, kWave, 0, 8><<<grid, kWave, 0, s>>>(a, w, p, g);
    else if (small) lp_policy_kernel<T, kWave, 0, 16><<<grid, kWave, 0, s>>>(a, w, p, g);
    else if (per <= 4) lp_policy_kernel<T, kRow, 0, 4><<<grid, kRow, 0, s>>>(a, w, p, g);
    else if (per <= 8) lp_policy_kernel<T, kRow, 0, 8><<<grid, kRow, 0, s>>>(a, w, p, g);
    else if (per <= 16) lp_policy_kernel<T, kRow, 0, 16><<<grid, kRow, 0, s>>>(a, w, p, g);
    else if (per <= 24) lp_policy_kernel<T, kRow, 8, 16><<<grid, kRow, 0, s>>>(a, w, p, g);
    else lp_policy_kernel<T, kRow, 8, 24><<<grid, kRow, 0, s>>>(a, w, p, g);
    lp_sum_kernel<<<1, 1024, 0, s>>>(w.row64, rows, g.sum);
    return true;
  }
  return false;
}

Rows make_rows(const void* x, int64_t xn, int64_t xs, int64_t n, int64_t s, int64_t v, const int64_t* target, int64_t tn,
               int64_t ts, int64_t ignore, double temperature) {
  const double k = temperature > 0.0 ? 1.4426950408889634074 / temperature : 0.0;
  return {x, xn, xs, target, tn, ts, n, s, v, ignore, (float)k, (float)(k - (double)(float)k)};
}

}  // namespace

extern "C" int64_t forge_logp_workspace(int dtype, int64_t n, int64_t s, int64_t v) {
  if (n <= 0 || dtype_size(dtype) == 0) return 16;
  // sequences of no tokens have counts and sums all the same
  return Layout(dtype, n, s > 0 ? s : 0, v > 0 ? v : 0).bytes;
}

extern "C" int forge_token_logps_fwd(int dtype, const void* logits, int64_t ld_n, int64_t ld_s, int64_t n, int64_t s,
                                     int64_t v, const int64_t* target, int64_t t_n, int64_t t_s, int64_t ignore_index,
                                     double temperature, float* logps, float* state, void* work, void* stream) {
  const Rows a = make_rows(logits, ld_n, ld_s, n, s, v, target, t_n, t_s, ignore_index, temperature);
  if (int rc = check_rows("token_logps_fwd", dtype, a, temperature)) return rc;
  if (n * s == 0) return FORGE_OK;
  if (int rc = check_given("token_logps_fwd", {logits, target, logps, work})) return rc;
  const Work w = Layout(dtype, n, s, v).work(work, logps, (float2*)state);
  hipStream_t st = (hipStream_t)stream;
  if (int rc = launch_partial(dtype, a, w, false, st)) return rc;
  return launch_rows(dtype, a, w, nullptr, st);
}

extern "C" int forge_token_logps_bwd(int dtype, const void* logits, int64_t ld_n, int64_t ld_s, int64_t n, int64_t s,
                                     int64_t v, const int64_t* target, int64_t t_n, int64_t t_s, int64_t ignore_index,
                                     double temperature, const float* logps, const float* state, const float* coef,
                                     int64_t c_n, int64_t c_s, const float* up, int64_t up_stride, int64_t up_count,
                                     void* dlogits, int64_t d_n, int64_t d_s, void* stream) {
  const Rows a = make_rows(logits, ld_n, ld_s, n, s, v, target, t_n, t_s, ignore_index, temperature);
  if (int rc = check_rows("token_logps_bwd", dtype, a, temperature)) return rc;
  if (n * s == 0) return FORGE_OK;
  if (int rc = check_given("token_logps_bwd", {logits, target, logps, state, coef, dlogits})) return rc;
  if (up && up_count <= 0) return forge_set_error(FORGE_ERR_INVALID, "token_logps_bwd: up_count %lld", (long long)up_count);
  const Grad g = {dlogits, d_n, d_s, coef, c_n, c_s, up, up_stride, up_count, (const float2*)state, logps,
                  (float)(1.0 / temperature), nullptr, nullptr};
  return launch_grad(dtype, a, g, true, (hipStream_t)stream);
}

extern "C" int forge_preference_fwd(int dtype, const void* logits, int64_t ld_n, int64_t ld_s, int64_t pairs, int64_t s,
                                    int64_t v, const int64_t* target, int64_t t_n, int64_t t_s, int64_t ignore_index,
                                    const float* ref, double beta, double label_smoothing, int kind, int normalized,
                                    int reduction, float* loss, float* seq_logps, float* rewards, float* coef,
                                    float* logps, float* state, void* work, void* stream) {
  const int64_t n = 2 * pairs;
  const Rows a = make_rows(logits, ld_n, ld_s, n, s, v, target, t_n, t_s, ignore_index, 1.0);
  if (int rc = check_rows("preference_fwd", dtype, a, 1.0)) return rc;
  if (kind != FORGE_PREF_SIGMOID && kind != FORGE_PREF_HINGE && kind != FORGE_PREF_IPO)
    return forge_set_error(FORGE_ERR_INVALID, "preference_fwd: kind %d", kind);
  if (reduction != FORGE_REDUCE_MEAN && reduction != FORGE_REDUCE_SUM && reduction != FORGE_REDUCE_NONE)
    return forge_set_error(FORGE_ERR_INVALID, "preference_fwd: reduction %d", reduction);
  if (pairs < 1) return forge_set_error(FORGE_ERR_INVALID, "preference_fwd: no pairs");
  if (int rc = check_given("preference_fwd", {loss, seq_logps, rewards, coef, work})) return rc;
  if (s > 0)
    if (int rc = check_given("preference_fwd", {logits, target, logps, state})) return rc;
  const Layout l(dtype, n, s, v);
  const Work w = l.work(work, logps, (float2*)state);
  double* seq = (double*)((char*)work + l.seq);
  hipStream_t st = (hipStream_t)stream;
  if (s > 0)
    if (int rc = launch_partial(dtype, a, w, false, st)) return rc;
  const int lanes = lanes_of(w.splits);
  if (int rc = by_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        lp_sequences_kernel<T><<<(unsigned)(n > kMaxGrid / 4 ? kMaxGrid / 4 : n), 1024, 0, st>>>(a, w, lanes, normalized != 0, seq);
      }))
    return rc;
  const Pairs p = {seq, w.counts, ref, pairs, beta, label_smoothing, kind, reduction, normalized != 0, loss, seq_logps,
                   rewards, coef};
  lp_pairs_kernel<<<1, kBlock, 0, st>>>(p);
  FORGE_CHECK_LAUNCH();
  return FORGE_OK;
}

extern "C" int forge_policy_loss_scaled(int dtype, const void* logits, int64_t ld_n, int64_t ld_s, int64_t n, int64_t s,
                                        int64_t v, const int64_t* target, int64_t t_n, int64_t t_s, int64_t ignore_index,
                                        double temperature, const float* advantages, int64_t a_n, int64_t a_s,
                                        const float* old_logps, int64_t o_n, int64_t o_s, const float* ref_logps,
                                        int64_t r_n, int64_t r_s, double clip_low, double clip_high, double kl_coef,
                                        int reduction, const float* grad_scale, float* loss, float* logps, float* kl,
                                        void* dlogits, int64_t d_n, int64_t d_s, void* work, void* stream) {
  const Rows a = make_rows(logits, ld_n, ld_s, n, s, v, target, t_n, t_s, ignore_index, temperature);
  if (int rc = check_rows("policy_loss", dtype, a, temperature)) return rc;
  if (reduction != FORGE_REDUCE_MEAN && reduction != FORGE_REDUCE_SUM && reduction != FORGE_REDUCE_SEQUENCE)
    return forge_set_error(FORGE_ERR_INVALID, "policy_loss: reduction %d", reduction);
  if (int rc = check_given("policy_loss", {loss, work})) return rc;
  if (n * s > 0)
    if (int rc = check_given("policy_loss", {logits, target, advantages, logps, kl})) return rc;
  const Layout l(dtype, n, s, v);
  const Work w = l.work(work, logps, (float2*)((char*)work + l.state));
  const Policy p = {advantages, a_n, a_s, old_logps, o_n, o_s, ref_logps, r_n, r_s, 1.0 - clip_low, 1.0 + clip_high,
                    kl_coef, reduction, kl, grad_scale};
  const Grad g = {dlogits, d_n, d_s, w.coef, s, 1, nullptr, 0, 1, w.state, logps, (float)(1.0 / temperature), w.row64, loss};
  hipStream_t st = (hipStream_t)stream;
  if (n * s > 0) {
    bool done = false;
    if (dlogits)
      if (int rc = by_dtype(dtype, [&](auto* t) { done = launch_policy<std::remove_pointer_t<decltype(t)>>(a, w, p, g, st); }))
        return rc;
    if (done) return FORGE_OK;
    if (int rc = launch_partial(dtype, a, w, true, st)) return rc;
    if (int rc = launch_rows(dtype, a, w, &p, st)) return rc;
  }
  return launch_grad(dtype, a, g, dlogits != nullptr && n * s > 0, st);
}

extern "C" int forge_policy_loss(int dtype, const void* logits, int64_t ld_n, int64_t ld_s, int64_t n, int64_t s, int64_t v,
                                 const int64_t* target, int64_t t_n, int64_t t_s, int64_t ignore_index,
                                 double temperature, const float* advantages, int64_t a_n, int64_t a_s,
                                 const float* old_logps, int64_t o_n, int64_t o_s, const float* ref_logps, int64_t r_n,
                                 int64_t r_s, double clip_low, double clip_high, double kl_coef, int reduction,
                                 float* loss, float* logps, float* kl, void* dlogits, int64_t d_n, int64_t d_s,
                                 void* work, void* stream) {
  return forge_policy_loss_scaled(dtype, logits, ld_n, ld_s, n, s, v, target, t_n, t_s, ignore_index, temperature,
                                  advantages, a_n, a_s, old_logps, o_n, o_s, ref_logps, r_n, r_s, clip_low, clip_high,
                                  kl_coef, reduction, nullptr, loss, logps, kl, dlogits, d_n, d_s, work, stream);
}
