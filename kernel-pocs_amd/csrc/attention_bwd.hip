// Attention backward for gfx950: three launches (four where there are few keys), no
// atomics (the sums have a fixed order).
//   -delta_i, delta_i = sum_d o_i dout_i, and -lse_i / scale, by head and query;
//   dq_i = scale sum_j ds_ij k_j,       a workgroup to 128 queries of a head;
//   dv_j = sum_i p_ij dout_i, dk_j = scale sum_i ds_ij q_i over the queries of the
//   group's heads,                      a workgroup to 128 keys of a kv head,
// with p_ij = exp2((s_ij - lse_i / scale) c), c = scale log2(e), computed again and
// ds_ij = p_ij (dout_i . v_j - delta_i).  p and ds are rounded to 16 bits as operands; every sum is in fp32.
// fp16 has few small values (2^-14 is the last with 11 bits), so there p is 2^14
// times as large, and ds times a power of two from 2^14 down to 1, a wave's choice that
// falls, with its sums, when one of its ds would pass fp16's largest value.  The sums
// are taken back at the end.  All of that is exact.
// 8 causal sequences, 16384 tokens in all, 32 heads of 128 on 8: 62 us (5.4 TB/s),
// 510 and 680 (both 960 TFLOP/s: matrix pipes and power, as in the forward).
// As in the forward, products are laid out so that p and ds stay in the
// registers that they are computed in: keys x queries for dq, queries x keys for
// dk and dv.
#include "attention.h"

namespace fattn {

template <class T>
constexpr float P_BITS = std::is_same_v<T, fp16_t> ? 14.f : 0.f;

// The wave's ds, 2^14 unit times what they are, within fp16's range as far as unit
// can fall; the sums follow.
template <class T, int DB>
__device__ __forceinline__ void keep_in_range(f32x16& ds, float& unit, f32x16 (&sums)[DB]) {
  if constexpr (std::is_same_v<T, fp16_t>) {
    while (true) {
      float top = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
      // (an infinite ds makes its own lane's sums so, whatever the unit)
      if (unit < 0x1p-13f || !__any(top > 65504.f && top < __builtin_inff())) return;
      unit *= 0.25f;
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] *= 0.25f;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) sums[db][r] *= 0.25f;
    }
  }
}

// whether a row has values that are not; by 16 lanes
template <class T>
__device__ __forceinline__ bool not_finite(const T* p, int D, int lane) {
  float t = 0.f;
#pragma unroll 1
  for (int d = lane % 16; d < D; d += 16) t = __builtin_fmaf(to_f32(p[d]), 0.f, t);
#pragma unroll
  for (int off = 8; off >= 1; off /= 2) t += __shfl_xor(t, off, 64);
  return t != t;
}

// rows [batch][row] of the query side, 16 lanes to a (row, head) at a time
template <class T>
__global__ __launch_bounds__(256) void attn_delta_kernel(Args a, float* shift, int64_t n_rows, int64_t pairs) {
  const int lane = threadIdx.x % 64;
  for (int64_t p = ((int64_t)blockIdx.x * 256 + threadIdx.x) / 16; p < pairs; p += (int64_t)gridDim.x * 16) {
    const int64_t row = p / a.H;
    const int head = (int)(p % a.H);
    const int64_t batch = a.cu_q ? 0 : row / a.tq, r = a.cu_q ? row : row % a.tq;
    const T* o = row_ptr<T>(a.o, batch, r, head);
    const T* d = row_ptr<T>(a.dout, batch, r, head);
    const float l = a.lse[p];
    float sum = 0.f;
    for (int c = 8 * (lane % 16); c < a.D; c += 128) {
      const Vec16<T> x = load16(o + c), y = load16(d + c);
      const uint2 low = *reinterpret_cast<const uint2*>(a.low + p * a.D + c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = to_f32(x.v[i]);
        sum += __builtin_fmaf((float)(int8_t)((i < 4 ? low.x : low.y) >> (8 * (i % 4))), low_step<T>(f), f) * to_f32(y.v[i]);
      }
    }
#pragma unroll
    for (int off = 8; off >= 1; off /= 2) sum += __shfl_xor(sum, off, 64);
    // The dk, dv kernel looks here for rows of q and dout that are not finite: the sum is
    // not where dout is not, nor where q is not, as o is NaN then.  But of a query without
    // keys o is 0, whatever it holds.
    if (l == -__builtin_inff() && a.causal && not_finite(row_ptr<T>(a.q, batch, r, head), a.D, lane)) sum = __builtin_nanf("");
    if (lane % 16 == 0) {
      a.delta[head * n_rows + row] = -sum;
      // a query without keys: exp(scale (s - inf)) = 0; one that sees scores of -inf alone
      // (o, and so the sum, is NaN): NaN, where it sees keys
      shift[head * n_rows + row] = l != -__builtin_inff() ? -l / a.scale : sum == sum ? l : sum;
    }
  }
}

template <class T, int DP>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attn_dq_kernel(Args a, const float* shift_of, int64_t n_rows, int tiles) {
  constexpr int BM = 128, BN = 64, KS = DP / 16, DB = DP / 32;
  using Dma = TileDma<DP, BN, 4>;
  __shared__ __attribute__((aligned(1024))) char smem[(DP == 256 ? 2 : 4) * Dma::BYTES];
  constexpr int NST = DP == 256 ? 1 : 2;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int G = a.H / a.Hkv, h = lane / 32;
  const Item it = item_of(blockIdx.x, tiles, a.Hkv, G);
  if (it.tile >= tiles) return;
  const LevelAt at = find_level(a.cu_q, a.B, a.tq, BM, it.tile);
  if (at.seq > a.B) return;
  const Span sq = span_of(a.cu_q, a.B, a.tq, at.seq);
  Span sk = span_of(a.cu_k, a.B, a.tk, at.seq);
  if (at.seq < 0 || at.seq >= a.B) sk.len = 0;
  const int head = it.kv * G + it.g;
  const int q0 = (at.level - 1) * BM;
  const int shift = sk.len - sq.len;
  const int rows = min(BM, sq.len - q0);
  const int k_end = a.causal ? min(sk.len, q0 + rows + shift) : sk.len;
  const int n_t = k_end > 0 ? (k_end + BN - 1) / BN : 0;
  const int wq = q0 + wave * 32, iq = wq + lane % 32;
  const bool live = iq < sq.len;
  bf16x8 qf[KS], df[KS];
  {
    const T* qp = row_ptr<T>(a.q, sq.batch, sq.start + (live ? iq : 0), head);
    const T* dp = row_ptr<T>(a.dout, sq.batch, sq.start + (live ? iq : 0), head);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = 16 * ks + 8 * h;
      uint4 v = make_uint4(0, 0, 0, 0), w = v;
      if (live && d < a.D) {
        v = *reinterpret_cast<const uint4*>(qp + d);
        w = *reinterpret_cast<const uint4*>(dp + d);
      }
      qf[ks] = __builtin_bit_cast(bf16x8, v);
      df[ks] = __builtin_bit_cast(bf16x8, w);
    }
  }
  const int64_t row = a.cu_q ? sq.start + iq : sq.batch * a.tq + iq;
  const float c = a.scale * LOG2E;
  const float below = live ? shift_of[head * n_rows + row] * c + P_BITS<T> : -__builtin_inff();
  float unit;
  const float delta = live ? a.delta[head * n_rows + row] : 0.f;

  Dma kd, vd;
  kd.setup(a.k.row, a.D);
  vd.setup(a.v.row, a.D);
  const T* kp = row_ptr<T>(a.k, sk.batch, sk.start, it.kv);
  const T* vp = row_ptr<T>(a.v, sk.batch, sk.start, it.kv);
  auto issue = [&](int t, int slot) {
    char* st = smem + slot * 2 * Dma::BYTES;
    kd.load(kp + (int64_t)t * BN * a.k.row, sk.len - t * BN, st, wave);
    vd.load(vp + (int64_t)t * BN * a.v.row, sk.len - t * BN, st + Dma::BYTES, wave);
  };
  RowFrag<DP> fr;
  ColFrag<DP> fc;
  fr.setup(lane);
  fc.setup(lane);
  f32x16 acc[DB];
  const int sees = a.causal ? min(sk.len, iq + shift + 1) : sk.len;
  const int all_see = a.causal ? min(sk.len, wq + shift + 1) : sk.len;
  const int any_sees = wq >= sq.len ? 0 : a.causal ? min(sk.len, min(wq + 32, sq.len) + shift) : sk.len;

  auto step = [&](int t, int slot, auto apart) __attribute__((always_inline)) {
    wait_dma<0>();
    barrier();
    if (NST == 2 && t + 1 < n_t) issue(t + 1, 1 - slot);
    char* kt = smem + slot * 2 * Dma::BYTES;
    const char* vt = kt + Dma::BYTES;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int k0 = t * BN + 32 * kb;
      if (!apart && k0 >= any_sees) continue;
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = mfma32<T>(fr.read(kt, 32 * kb, ks), qf[ks], s);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) dp = mfma32<T>(fr.read(vt, 32 * kb, ks), df[ks], dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = exp2_hw(__builtin_fmaf(s[r], c, below)) * ((dp[r] + delta) * unit);
      if (k0 + 32 > all_see) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 8 * (r / 4) + 4 * h + r % 4 >= sees) s[r] = 0.f;
      }
      keep_in_range<T>(s, unit, acc);
      if constexpr (apart) {  // (the sign of ds is not known: NaN)
        __syncthreads();        // every wave has its scores of these keys
        Special<T, DP>::add(acc, kt, 32 * kb, 32, k0, 0, sees, true);
        __syncthreads();
        Special<T, DP>::clear(kt, 32 * kb, 32, wave, 4);
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bf16x8 ds = pack_acc<T>(s, i);
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = mfma32<T>(fc.read(kt, 32 * kb + 16 * i, db), ds, acc[db]);
      }
    }
    if (NST == 1 && t + 1 < n_t) {
      wait_dma<0>();
      barrier();  // every wave has read the tile
      issue(t + 1, 0);
    }
  };
  auto run = [&](auto apart) __attribute__((always_inline)) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;
    unit = 1.f;
    if (n_t > 0) issue(0, 0);
    for (int t = 0; t < n_t; t += NST) {
      step(t, 0, apart);
      if (NST == 2 && t + 1 < n_t) step(t + 1, 1, apart);
    }
  };
  run(std::false_type());
  if (a.causal && any_of_4_waves(smem, wave, any_nan(acc))) run(std::true_type());
  if (!live) return;
  const float back = a.scale * exp2f(-P_BITS<T>) / unit;
  T* op = row_ptr<T>(a.dq, sq.batch, sq.start + iq, head);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * db + 8 * i + 4 * h;
      if (d >= a.D) continue;
      store4(op + d, acc[db][4 * i] * back, acc[db][4 * i + 1] * back, acc[db][4 * i + 2] * back,
             acc[db][4 * i + 3] * back);
    }
}

// A wave keeps 32 keys and values (the products' second operands) and their
// gradients in registers: one wave a SIMD.  At DP = 256 those take more registers
// than there are, so dk and dv are a launch each (DK, DV).
template <class T, int DP, bool DK, bool DV>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attn_dkv_kernel(Args a, const float* shift_of, int64_t n_rows, int tiles) {
  constexpr int BN = 128, BQ = DP == 256 ? 32 : 64, KS = DP / 16, DB = DP / 32;
  using Dma = TileDma<DP, BQ, 4>;
  // One array: beside a second one the compiler waits for all LDS-DMA before it
  // reads.  -lse / scale and -delta of two slots come first, the tiles TILES behind
  // them, which is part of the fragments' bases: their immediates reach 64 KB.
  constexpr int TILES = 1024;
  __shared__ __attribute__((aligned(1024))) char smem[TILES + 2 * 2 * Dma::BYTES];
  auto stat = [&](int slot, int i) __attribute__((always_inline)) { return reinterpret_cast<float*>(smem) + (slot * 2 + i) * 64; };
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int G = a.H / a.Hkv, h = lane / 32;
  const Item it = item_of(blockIdx.x, tiles, a.Hkv, a.parts);
  if (it.tile >= tiles) return;
  const LevelAt at = find_level(a.cu_k, a.B, a.tk, BN, it.tile);
  if (at.seq > a.B) return;
  const Span sk = span_of(a.cu_k, a.B, a.tk, at.seq);
  Span sq = span_of(a.cu_q, a.B, a.tq, at.seq);
  if (at.seq < 0 || at.seq >= a.B) sq.len = 0;
  const int k0 = ((sk.len + BN - 1) / BN - at.level) * BN, wk = k0 + wave * 32, jk = wk + lane % 32;
  const bool live = jk < sk.len;
  const int shift = sk.len - sq.len;
  bf16x8 kf[KS], vf[KS];
  {
    const T* kp = row_ptr<T>(a.k, sk.batch, sk.start + (live ? jk : 0), it.kv);
    const T* vp = row_ptr<T>(a.v, sk.batch, sk.start + (live ? jk : 0), it.kv);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = 16 * ks + 8 * h;
      uint4 v = make_uint4(0, 0, 0, 0), w = v;
      if (live && d < a.D) {
        v = *reinterpret_cast<const uint4*>(kp + d);
        w = *reinterpret_cast<const uint4*>(vp + d);
      }
      kf[ks] = __builtin_bit_cast(bf16x8, v);
      vf[ks] = __builtin_bit_cast(bf16x8, w);
    }
  }
  // the first query that sees a key of the tile, and tiles of queries from there, of
  // each of the group's heads in turn
  const int first = a.causal ? max(0, k0 - shift) / BQ * BQ : 0;
  const int g_lo = G * it.g / a.parts, g_hi = G * (it.g + 1) / a.parts;  // of this part
  const int n_t = sq.len > first ? (sq.len - first + BQ - 1) / BQ * (g_hi - g_lo) : 0;
  Dma qd, dd;
  qd.setup(a.q.row, a.D);
  dd.setup(a.dout.row, a.D);
  int next_i = first, next_head = it.kv * G + g_lo;  // of the tile that is issued next
  auto issue = [&](int slot) {
    const int left = sq.len - next_i;
    char* st = smem + TILES + slot * 2 * Dma::BYTES;
    qd.load(row_ptr<T>(a.q, sq.batch, sq.start + next_i, next_head), left, st, wave);
    dd.load(row_ptr<T>(a.dout, sq.batch, sq.start + next_i, next_head), left, st + Dma::BYTES, wave);
    // (rows that do not exist: q = dout = 0, so p = exp2(0) and ds = 0 add zeros)
    const int64_t row = (a.cu_q ? sq.start : sq.batch * a.tq) + next_i;
    if (wave < 2) {
      const __amdgpu_buffer_rsrc_t r = make_rsrc((wave ? a.delta : shift_of) + next_head * n_rows + row);
      dma4(r, stat(slot, wave), lane < left && lane < BQ ? lane * 4 : OOB);
    }
    next_i += BQ;
    if (next_i >= sq.len) {
      next_i = first;
      ++next_head;
    }
  };
  RowFrag<DP> fr;
  ColFrag<DP> fc;
  fr.setup(lane);
  fc.setup(lane);
  for (int& x : fr.base) asm("" : "+v"(x += TILES));
  for (int& x : fc.base) asm("" : "+v"(x += TILES));
  // Whether a query that sees some of these keys and not all, or is in a tile with such
  // (from `first` on), has a q or dout that is not finite (delta tells): its p and ds of
  // the others are 0, but their products with it are NaN.
  bool odd = false;
  if (a.causal && n_t > 0) {
    const int n = min(sq.len, k0 + BN - 1 - shift) - first;
    const int64_t row = (a.cu_q ? sq.start : sq.batch * a.tq) + first;
    for (int head = it.kv * G + g_lo; head < it.kv * G + g_hi; ++head)
      for (int i = threadIdx.x; i < n; i += 256) odd |= !__builtin_isfinite(a.delta[head * n_rows + row + i]);
  }
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[db][r] = dv[db][r] = 0.f;
  const float c = a.scale * LOG2E;
  float unit = 1.f;

  int tile_i = first;
  auto step = [&](bool more, int slot, auto apart, auto on_k, auto on_v) __attribute__((always_inline)) {
    wait_dma<0>();
    barrier();
    if (more) issue(1 - slot);
    const int t_i = tile_i;
    tile_i = tile_i + BQ < sq.len ? tile_i + BQ : first;
    char* qt = smem + slot * 2 * Dma::BYTES;
    char* dt = qt + Dma::BYTES;
#pragma unroll
    for (int qb = 0; qb < BQ / 32; ++qb) {
      __builtin_amdgcn_sched_barrier(0);
      const int i0 = t_i + 32 * qb;
      // (causal: the last query of the block sees nothing of this wave's keys)
      if (i0 >= sq.len || (!apart && (wk >= sk.len || (a.causal && i0 + 31 + shift < wk)))) continue;
      f32x16 s, dp;  // begin with -lse / scale and -delta of their queries
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(stat(slot, 0) + 32 * qb + 8 * i + 4 * h);
        const f32x4 y = *reinterpret_cast<const f32x4*>(stat(slot, 1) + 32 * qb + 8 * i + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[4 * i + j] = x[j];
          dp[4 * i + j] = y[j];
        }
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = mfma32<T>(fr.read(qt, 32 * qb, ks), kf[ks], s);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        if constexpr (on_k) dp = mfma32<T>(fr.read(dt, 32 * qb, ks), vf[ks], dp);
      if (a.causal && i0 + shift < wk + 31) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (i0 + 8 * (r / 4) + 4 * h + r % 4 + shift < jk) {
            s[r] = -__builtin_inff();
            dp[r] = 0.f;
          }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = exp2_hw(P_BITS<T> ? __builtin_fmaf(s[r], c, P_BITS<T>) : s[r] * c);
        dp[r] *= s[r] * unit;
      }
      if constexpr (on_k) keep_in_range<T>(dp, unit, dk);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (apart) {  // (the fragments read the tiles TILES behind qt and dt)
        __syncthreads();      // every wave has its scores of these queries
        if constexpr (on_k) Special<T, DP>::add(dk, qt + TILES, 32 * qb, 32, i0, jk - shift, sq.len, true);
        if constexpr (on_v) Special<T, DP>::add(dv, dt + TILES, 32 * qb, 32, i0, jk - shift, sq.len, false);
        __syncthreads();
        if constexpr (on_k) Special<T, DP>::clear(qt + TILES, 32 * qb, 32, wave, 4);
        if constexpr (on_v) Special<T, DP>::clear(dt + TILES, 32 * qb, 32, wave, 4);
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bf16x8 p = pack_acc<T>(s, i), ds = pack_acc<T>(dp, i);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          if constexpr (on_v) dv[db] = mfma32<T>(fc.read(dt, 32 * qb + 16 * i, db), p, dv[db]);
          if constexpr (on_k) dk[db] = mfma32<T>(fc.read(qt, 32 * qb + 16 * i, db), ds, dk[db]);
        }
      }
    }
  };
  auto store = [&](auto on_k, auto on_v) __attribute__((always_inline)) {
    if (!live) return;
    const float p_one = exp2f(-P_BITS<T>), back = a.scale * p_one / unit;
    if (a.parts > 1) {
      const int64_t n_k = a.cu_k ? a.tk : a.tk * a.B, row = (a.cu_k ? sk.start : sk.batch * a.tk) + jk;
      float* p = a.part + ((it.g * n_k + row) * a.Hkv + it.kv) * 2 * a.D;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = 32 * db + 8 * i + 4 * h;
          if (d >= a.D) continue;
          if constexpr (on_k)
            *reinterpret_cast<f32x4*>(p + d) = f32x4{dk[db][4 * i], dk[db][4 * i + 1], dk[db][4 * i + 2], dk[db][4 * i + 3]} * back;
          if constexpr (on_v)
            *reinterpret_cast<f32x4*>(p + a.D + d) = f32x4{dv[db][4 * i], dv[db][4 * i + 1], dv[db][4 * i + 2], dv[db][4 * i + 3]} * p_one;
        }
      return;
    }
    T* kp = row_ptr<T>(a.dk, sk.batch, sk.start + jk, it.kv);
    T* vp = row_ptr<T>(a.dv, sk.batch, sk.start + jk, it.kv);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * db + 8 * i + 4 * h;
        if (d >= a.D) continue;
        if constexpr (on_k)
          store4(kp + d, dk[db][4 * i] * back, dk[db][4 * i + 1] * back, dk[db][4 * i + 2] * back,
                 dk[db][4 * i + 3] * back);
        if constexpr (on_v) store4(vp + d, dv[db][4 * i] * p_one, dv[db][4 * i + 1] * p_one, dv[db][4 * i + 2] * p_one, dv[db][4 * i + 3] * p_one);
      }
  };
  typedef std::bool_constant<DK> WithK;
  typedef std::bool_constant<DV> WithV;
  if (n_t > 0) issue(0);
  // (through slot 1's statistics, which are not under way yet)
  if (a.causal && any_of_4_waves(smem + TILES / 2, wave, odd)) {
    // dk and dv one after the other: together they take more registers than there are
    auto pass = [&](auto on_k, auto on_v) __attribute__((always_inline)) {
      tile_i = next_i = first;
      next_head = it.kv * G + g_lo;
      __syncthreads();
      if (n_t > 0) issue(0);
#pragma unroll 1
      for (int t = 0; t < n_t; ++t) step(t + 1 < n_t, t % 2, std::true_type(), on_k, on_v);
      store(on_k, on_v);
    };
    if constexpr (DK) pass(WithK(), std::false_type());
    if constexpr (DV) pass(std::false_type(), WithV());
    return;
  }
  for (int t = 0; t < n_t; t += 2) {
    step(t + 1 < n_t, 0, std::false_type(), WithK(), WithV());
    if (t + 1 < n_t) step(t + 2 < n_t, 1, std::false_type(), WithK(), WithV());
  }
  store(WithK(), WithV());
}

// dk and dv: the sums of the parts, in order.  4 values a thread.
template <class T>
__global__ __launch_bounds__(256) void attn_dkv_join_kernel(Args a, int64_t n_k) {
  const int vecs = a.D / 4;
  const int64_t n = n_k * a.Hkv * 2 * vecs;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < n; x += (int64_t)gridDim.x * 256) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < a.parts; ++p) v += *reinterpret_cast<const f32x4*>(a.part + (p * n + x) * 4);
    const int d = (int)(x % vecs) * 4, which = (int)(x / vecs % 2), head = (int)(x / vecs / 2 % a.Hkv);
    const int64_t row = x / vecs / 2 / a.Hkv, batch = a.cu_k ? 0 : row / a.tk;
    store4(row_ptr<T>(which ? a.dv : a.dk, batch, a.cu_k ? row : row % a.tk, head) + d, v[0], v[1], v[2], v[3]);
  }
}

// Parts of a group's heads, a workgroup each (13 sequences of 3001 tokens, 14 heads of 64
// on 2: 80 workgroups 84 us, 480 35 and 5 for the join): where the tiles of keys alone would
// leave CUs without work (two workgroups a CU are resident), and where a
// workgroup has at least 16 tiles of queries to go through (a tile takes longer than
// its share of the join).
int dkv_parts(const Args& a) {
  const int64_t G = a.H / a.Hkv, wgs = most_tiles(a.cu_k, a.B, a.tk, 128) * a.Hkv;
  const int64_t queries = a.cu_q ? a.tq / (a.B > 0 ? a.B : 1) : a.tq;  // of a sequence
  if (wgs == 0 || G * queries < 16 * 64) return 1;
  const int64_t parts = 512 / wgs;
  return (int)(parts < 1 ? 1 : parts > G ? G : parts);
}

template <class T, int DP, bool DK, bool DV>
static int launch_dkv(const Args& a, const float* shift, int64_t n_rows, int64_t n, int64_t tiles, hipStream_t s) {
  attn_dkv_kernel<T, DP, DK, DV><<<(unsigned)n, 256, 0, s>>>(a, shift, n_rows, (int)tiles);
  FORGE_CHECK_LAUNCH();
  return FORGE_OK;
}

template <class T, int DP>
static int launch_bwd_dp(const Args& a, float* shift, int64_t n_rows, hipStream_t s) {
  const int64_t tq = most_tiles(a.cu_q, a.B, a.tq, 128), tk = most_tiles(a.cu_k, a.B, a.tk, 128);
  const int64_t nq = items(tq, a.Hkv, a.H / a.Hkv), nk = items(tk, a.Hkv, a.parts);
  if (nq > 0x7fffffffLL || nk > 0x7fffffffLL) return forge_set_error(FORGE_ERR_INVALID, "attention: too many tiles");
  const int64_t pairs = n_rows * a.H;
  if (pairs) attn_delta_kernel<T><<<grid_for(pairs * 16, 256, 256 * 64), 256, 0, s>>>(a, shift, n_rows, pairs);
  FORGE_CHECK_LAUNCH();
  if (nq && n_rows) attn_dq_kernel<T, DP><<<(unsigned)nq, 256, 0, s>>>(a, shift, n_rows, (int)tq);
  FORGE_CHECK_LAUNCH();
  if (nk == 0) return FORGE_OK;
  if (int e = launch_dkv<T, DP, true, DP < 256>(a, shift, n_rows, nk, tk, s)) return e;
  if (DP == 256)
    if (int e = launch_dkv<T, DP, DP < 256, true>(a, shift, n_rows, nk, tk, s)) return e;
  if (a.parts > 1) {
    const int64_t n_k = a.cu_k ? a.tk : a.tk * a.B;
    attn_dkv_join_kernel<T><<<grid_for(n_k * a.Hkv * 2 * (a.D / 4), 256, 256 * 16), 256, 0, s>>>(a, n_k);
    FORGE_CHECK_LAUNCH();
  }
  return FORGE_OK;
}

template <class T>
static int launch_bwd_t(const Args& a, float* shift, int64_t n_rows, hipStream_t s) {
  if (a.D <= 64) return launch_bwd_dp<T, 64>(a, shift, n_rows, s);
  if (a.D <= 128) return launch_bwd_dp<T, 128>(a, shift, n_rows, s);
  return launch_bwd_dp<T, 256>(a, shift, n_rows, s);
}

int launch_bwd(int dtype, const Args& a, float* shift, int64_t n_rows, hipStream_t s) {
  return dtype == FORGE_DTYPE_F16 ? launch_bwd_t<fp16_t>(a, shift, n_rows, s) : launch_bwd_t<bf16_t>(a, shift, n_rows, s);
}

}  // namespace fattn
