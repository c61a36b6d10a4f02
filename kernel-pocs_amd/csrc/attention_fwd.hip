// Attention forward for gfx950.
//
// One pass over the keys with a running maximum m and sum l a query:
//   S^T = K Q^T (keys x queries), p = exp2(s c - m) with c = scale log2(e),
//   O^T += V^T P^T, and at the end o = O / l, lse = (m + log2 l) ln 2.
// Both products are formed transposed, so that a lane of v_mfma_f32_32x32x16
// holds one query's scores (the maximum and the sum are in-lane, with one exchange
// between the halves of the wave), and those registers, rounded to 16 bits,
// are the second product's operand as they are: P never leaves registers.
// Rounding p to 16 bits errs by half a step of each term at random, less than
// the rounding of the result.
//
// A workgroup of 4 waves takes 128 queries of one head, 32 a wave; tiles of 64
// keys and values come by LDS-DMA into a ring of two.  8 causal sequences, 16384
// tokens, 32 heads of 128 on 8: 390 to 410 us, 820 TFLOP/s.  Of its parts MFMA alone
// reaches 1680, with LDS-DMA and barriers 1270, with the reads of LDS 1020: each wave
// reads all of a tile for itself, 1024 cycles of LDS beside 1031 of MFMA, and the softmax
// stands between its two products (power adds to that: 1150 where the data are
// zeros).  8 waves to 256 queries, or 64 queries a wave, were slower (870 and 754 where
// this ran 890).
#include "attention.h"

namespace fattn {

constexpr int BN = 64;
constexpr float SLACK = 6.f;

template <class T, int DP>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attn_fwd_kernel(Args a, int tiles) {
  constexpr int BM = 128, KS = DP / 16, DB = DP / 32;
  using Dma = TileDma<DP, BN, 4>;
  __shared__ __attribute__((aligned(1024))) char smem[4 * Dma::BYTES];
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

  const int wq = q0 + wave * 32, iq = wq + lane % 32;  // this wave's first query, this lane's
  const bool live = iq < sq.len;
  bf16x8 qf[KS];
  {
    const T* qp = row_ptr<T>(a.q, sq.batch, sq.start + (live ? iq : 0), head);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = 16 * ks + 8 * h;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (live && d < a.D) v = *reinterpret_cast<const uint4*>(qp + d);
      qf[ks] = __builtin_bit_cast(bf16x8, v);
    }
  }
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

  f32x16 o[DB];
  const float c = a.scale * LOG2E;
  float m, l;  // m: the maximum less P_UP, in units of log2; l: this half's sum
  float down = 1.f;  // of the values, in the second run

  // keys that this lane's query sees, and those that every query of the wave does
  const int sees = a.causal ? min(sk.len, iq + shift + 1) : sk.len;
  const int all_see = a.causal ? min(sk.len, wq + shift + 1) : sk.len;
  const int any_sees = wq >= sq.len ? 0 : a.causal ? min(sk.len, min(wq + 32, sq.len) + shift) : sk.len;

  // (slot: a constant where the call is, so that it is part of the reads' immediates)
  auto step = [&](int t, int slot, auto apart) __attribute__((always_inline)) {
    wait_dma<0>();
    barrier();
    if (t + 1 < n_t) issue(t + 1, 1 - slot);
    const int k0 = t * BN;
    if (!apart && k0 >= any_sees) return;
    const char* kt = smem + slot * 2 * Dma::BYTES;
    char* vt = smem + slot * 2 * Dma::BYTES + Dma::BYTES;
    f32x16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[kb] = mfma32<T>(fr.read(kt, 32 * kb, ks), qf[ks], s[kb]);
    }
    if (k0 + BN > all_see) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 32 * kb + 8 * (r / 4) + 4 * h + r % 4 >= sees) s[kb][r] = -__builtin_inff();
    }
    float top = s[0][0];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
    top = __builtin_fmaf(fmaxf(top, other_half(top)), c, -P_UP<T>);
    // m follows the maximum by steps of SLACK at least: p stays below 2^(SLACK + P_UP), and
    // the sums are seldom scaled (a new maximum, however small, comes up in one of
    // 32 queries at almost every tile)
    if (__any(top > m + SLACK)) {
      const float up = top > m + SLACK ? top : m, f = exp2_hw(m - up);
      m = up;
      l *= f;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= f;
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = exp2_hw(__builtin_fmaf(s[kb][r], c, -m));
        l += p;
        s[kb][r] = p;
      }
    if constexpr (apart) {
      Special<T, DP>::add(o, vt, 0, BN, k0, 0, sees, false);
      __syncthreads();
      Special<T, DP>::clear(vt, 0, BN, wave, 4, down);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bf16x8 p = pack_acc<T>(s[i / 2], i % 2);
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = mfma32<T>(fc.read(vt, 16 * i, db), p, o[db]);
    }
  };
  auto run = [&](auto apart) __attribute__((always_inline)) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
    m = -__FLT_MAX__;
    l = 0.f;
    if (n_t > 0) issue(0, 0);
    for (int t = 0; t < n_t; t += 2) {
      step(t, 0, apart);
      if (t + 1 < n_t) step(t + 1, 1, apart);
    }
  };
  run(std::false_type());
  if (second_run<T>(a.causal) && any_of_4_waves(smem, wave, any_nan(o))) {
    down = v_down<T>(sk.len);
    run(std::true_type());
  }
  l += other_half(l);
  if (!live) return;
  const float inv = l == 0.f ? nothing(sees) : 1.f / (l * down);
  T* op = row_ptr<T>(a.o, sq.batch, sq.start + iq, head);
  const int64_t row = a.cu_q ? sq.start + iq : sq.batch * a.tq + iq;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * db + 8 * i + 4 * h;
      if (d >= a.D) continue;
      store4(op + d, o[db][4 * i] * inv, o[db][4 * i + 1] * inv, o[db][4 * i + 2] * inv, o[db][4 * i + 3] * inv);
      if (a.low)
        store_low4<T>(a.low + (row * a.H + head) * a.D + d, o[db][4 * i] * inv, o[db][4 * i + 1] * inv, o[db][4 * i + 2] * inv,
                      o[db][4 * i + 3] * inv);
    }
  if (h == 0 && a.lse) a.lse[row * a.H + head] = l == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * LN2;
}

template <class T, int DP>
static int launch_fwd_dp(const Args& a, hipStream_t s) {
  const int64_t tiles = most_tiles(a.cu_q, a.B, a.tq, 128);
  const int64_t n = items(tiles, a.Hkv, a.H / a.Hkv);
  if (n > 0x7fffffffLL) return forge_set_error(FORGE_ERR_INVALID, "attention: too many tiles");
  if (n == 0) return FORGE_OK;
  attn_fwd_kernel<T, DP><<<(unsigned)n, 256, 0, s>>>(a, (int)tiles);
  FORGE_CHECK_LAUNCH();
  return FORGE_OK;
}

template <class T>
static int launch_fwd_t(const Args& a, hipStream_t s) {
  if (a.D <= 64) return launch_fwd_dp<T, 64>(a, s);
  if (a.D <= 128) return launch_fwd_dp<T, 128>(a, s);
  return launch_fwd_dp<T, 256>(a, s);
}

int launch_fwd(int dtype, const Args& a, hipStream_t s) {
  return dtype == FORGE_DTYPE_F16 ? launch_fwd_t<fp16_t>(a, s) : launch_fwd_t<bf16_t>(a, s);
}

}  // namespace fattn
