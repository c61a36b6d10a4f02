// Attention of few queries a sequence (a serving step: one token each) for
// gfx950.  Keys and values are read once and set the time.
//
// The queries of a group's heads share a kv head: they are the rows t G + g of
// one tile of 32 (t: token, g: head), the second operand of the same products
// as in attention_fwd.hip.  The keys of a sequence are cut into chunks of C
// (a multiple of the waves' 32), a workgroup to a chunk and kv head, so that a long
// cache is read by many CUs; its waves take 32 keys in turn, each through an LDS
// ring of its own, without barriers.  The waves' sums are joined in LDS; those of
// several chunks by a second launch.  Every sum has a fixed order.
//
// 32 sequences of 131072 keys in all, 8 kv heads of 128, a token each: 106 us, keys and
// values at 5.1 TB/s, and 6 for the join.  4 tokens and 2004 keys: 9 and 5 us.
#include "attention.h"

namespace fattn {

struct Parts {      // of a chunk: [chunk of its sequence][query * H + head]
  float* o;         // [D], its output (divided by its sum)
  float* m;         // maximum less P_UP, in units of log2
  float* l;         // sum of p, relative to 2^m
  int64_t n;        // queries * H
  int C;            // keys a chunk
};

__device__ __forceinline__ int chunks_of(int len, int C) { return max(1, (len + C - 1) / C); }

template <class T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, 1) void attn_rows_kernel(Args a, Parts parts) {
  constexpr int KS = DP / 16, DB = DP / 32, PITCH = DP + 4;
  using Dma = TileDma<DP, 32, 1>;
  constexpr int RING = NW * 2 * 2 * Dma::BYTES, SUMS = NW * 32 * PITCH * 4;
  // (one array: beside a second one the compiler waits for all LDS-DMA before it reads)
  constexpr int STAT = RING > SUMS ? RING : SUMS;
  __shared__ __attribute__((aligned(1024))) char smem[STAT + 3 * NW * 32 * 4];
  float* const stat = reinterpret_cast<float*>(smem + STAT);  // [3][NW][32]: maxima, sums of p, 1 / down
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), h = lane / 32;
  const int G = a.H / a.Hkv, kv = blockIdx.y;
  const TileAt at = find_tile(a.cu_k, a.B, a.tk, parts.C, blockIdx.x, 1);
  if (at.seq > a.B) return;
  // (rows before the first offset or behind the last: each side without the other)
  const bool inside = at.seq >= 0 && at.seq < a.B;
  const Span sq = span_of(a.cu_q, a.B, a.tq, at.seq);
  Span sk = span_of(a.cu_k, a.B, a.tk, at.seq);
  if (!inside) {
    if (at.tile > 0) return;
    sk.len = 0;
  }
  const int n_chunk = chunks_of(sk.len, parts.C), lo = at.tile * parts.C, hi = min(sk.len, lo + parts.C);
  const int n_rows = sq.len * G, shift = sk.len - sq.len;
  const float c = a.scale * LOG2E;
  Dma kd, vd;
  kd.setup(a.k.row, a.D);
  vd.setup(a.v.row, a.D);
  const T* kp = row_ptr<T>(a.k, sk.batch, sk.start, kv);
  const T* vp = row_ptr<T>(a.v, sk.batch, sk.start, kv);
  char* ring = smem + wave * 2 * 2 * Dma::BYTES;
  RowFrag<DP> fr;
  ColFrag<DP> fc;
  fr.setup(lane);
  fc.setup(lane);
  const int n_t = hi > lo ? (hi - lo + 31) / 32 : 0, mine = n_t > wave ? (n_t - wave + NW - 1) / NW : 0;
  auto issue = [&](int i) {
    const int k0 = lo + 32 * (wave + i * NW);
    char* st = ring + (i % 2) * 2 * Dma::BYTES;
    kd.load(kp + (int64_t)k0 * a.k.row, sk.len - k0, st, 0);
    vd.load(vp + (int64_t)k0 * a.v.row, sk.len - k0, st + Dma::BYTES, 0);
  };

  for (int r0 = 0; r0 < n_rows; r0 += 32) {
    const int row = r0 + lane % 32, token = row / G, head = kv * G + row % G;
    const bool live = row < n_rows;
    if (mine > 0) issue(0);
    if (mine > 1) issue(1);
    bf16x8 qf[KS];
    const T* qp = row_ptr<T>(a.q, sq.batch, sq.start + (live ? token : 0), head);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = 16 * ks + 8 * h;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (live && d < a.D) v = *reinterpret_cast<const uint4*>(qp + d);
      qf[ks] = __builtin_bit_cast(bf16x8, v);
    }
    f32x16 o[DB];
    float m, l, down = 1.f;  // down: of the values, in the second run
    const int sees = a.causal ? min(sk.len, token + shift + 1) : sk.len;
    auto run = [&](auto apart) __attribute__((always_inline)) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
      m = -__FLT_MAX__;
      l = 0.f;
      for (int i = 0; i < mine; ++i) {
        if (i + 1 < mine) wait_dma<2 * Dma::N>();
        else wait_dma<0>();
        const int k0 = lo + 32 * (wave + i * NW);
        const char* kt = ring + (i % 2) * 2 * Dma::BYTES;
        char* vt = ring + (i % 2) * 2 * Dma::BYTES + Dma::BYTES;
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = mfma32<T>(fr.read(kt, 0, ks), qf[ks], s);
        float top = -__builtin_inff();
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (k0 + 8 * (r / 4) + 4 * h + r % 4 >= sees) s[r] = -__builtin_inff();
          top = fmaxf(top, s[r]);
        }
        top = __builtin_fmaf(fmaxf(top, other_half(top)), c, -P_UP<T>);
        const float up = fmaxf(top, m), f = exp2_hw(m - up);
        m = up;
        l *= f;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[db][r] *= f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = exp2_hw(__builtin_fmaf(s[r], c, -m));
          l += s[r];
        }
        if constexpr (apart) {  // (the wave's own ring; its LDS accesses keep their order)
          Special<T, DP>::add(o, vt, 0, 32, k0, 0, sees, false);
          Special<T, DP>::clear(vt, 0, 32, 0, 1, down);
          wait_dma<0>();
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bf16x8 p = pack_acc<T>(s, j);
#pragma unroll
          for (int db = 0; db < DB; ++db) o[db] = mfma32<T>(fc.read(vt, 16 * j, db), p, o[db]);
        }
        wait_dma<2 * Dma::N>();  // (the reads of this slot are done; the other slot's DMA may be under way)
        if (i + 2 < mine) issue(i + 2);
      }
    };
    run(std::false_type());
    if (second_run<T>(a.causal && sq.len > 1) && mine > 0 && __any(any_nan(o))) {  // (a token alone sees every key)
      down = v_down<T>(sk.len);
      wait_dma<0>();  // the reads of the ring are done
      issue(0);
      if (mine > 1) issue(1);
      run(std::true_type());
    }
    l += other_half(l);
    wait_dma<0>();
    barrier();  // every wave is done with its ring
    float* sums = reinterpret_cast<float*>(smem) + wave * 32 * PITCH + (lane % 32) * PITCH;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(sums + 32 * db + 8 * i + 4 * h) =
            f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
    if (h == 0) {
      stat[wave * 32 + lane] = m;
      stat[(NW + wave) * 32 + lane] = l;
      stat[(2 * NW + wave) * 32 + lane] = 1.f / down;
    }
    __syncthreads();
    const int rows = min(32, n_rows - r0), vecs = a.D / 4;
    for (int x = threadIdx.x; x < rows * vecs; x += NW * 64) {
      const int r = x / vecs, d = x % vecs * 4, t = (r0 + r) / G, hd = kv * G + (r0 + r) % G;
      float top = stat[r];
#pragma unroll
      for (int w = 1; w < NW; ++w) top = fmaxf(top, stat[w * 32 + r]);
      // (divided by the sum first: the waves' sums may be past fp32's range together, or
      // without their factors)
      float total = 0.f, f[NW], v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        f[w] = exp2_hw(stat[w * 32 + r] - top);
        total += stat[(NW + w) * 32 + r] * f[w];
        f[w] *= stat[(2 * NW + w) * 32 + r];
      }
      // (of a chunk of several 0: the join looks at them all)
      const float inv = total != 0.f ? 1.f / total : n_chunk == 1 ? nothing(a.causal ? min(sk.len, t + shift + 1) : sk.len) : 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(smem) + (w * 32 + r) * PITCH + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += y[j] * (f[w] * inv);
      }
      const int64_t q = (a.cu_q ? sq.start : sq.batch * a.tq) + t;
      if (n_chunk == 1) {
        store4(row_ptr<T>(a.o, sq.batch, sq.start + t, hd) + d, v[0], v[1], v[2], v[3]);
        if (a.low) store_low4<T>(a.low + (q * a.H + hd) * a.D + d, v[0], v[1], v[2], v[3]);
        if (d == 0 && a.lse) a.lse[q * a.H + hd] = total == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(total)) * LN2;
      } else {
        const int64_t at_part = at.tile * parts.n + q * a.H + hd;
        *reinterpret_cast<f32x4*>(parts.o + at_part * a.D + d) = f32x4{v[0], v[1], v[2], v[3]};
        if (d == 0) {
          parts.m[at_part] = top;
          parts.l[at_part] = total;
        }
      }
    }
    __syncthreads();
  }
}

// Joins the chunks of sequences that have several: a wave to a (query, head).
template <class T>
__global__ __launch_bounds__(256) void attn_join_kernel(Args a, Parts parts) {
  const int lane = threadIdx.x % 64;
  const int64_t p = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (p >= parts.n) return;
  const int64_t q = p / a.H;
  const int head = (int)(p % a.H);
  Span sk = {0, 0, 0};
  int64_t batch = 0, row = q;
  int behind = 0;  // queries of the sequence behind this one
  if (!a.cu_q) {
    batch = q / a.tq;
    row = q % a.tq;
    sk = span_of(nullptr, a.B, a.tk, (int)batch);
    behind = (int)(a.tq - 1 - row);
  } else {
    for (int base = 0; base < a.B; base += 64) {
      const int s = base + lane;
      Span sq = {0, 0, 0};
      if (s < a.B) sq = span_of(a.cu_q, a.B, a.tq, s);
      const uint64_t found = __ballot(q >= sq.start && q < sq.start + sq.len);
      if (found) {
        const int at = __builtin_ctzll(found);
        sk = span_of(a.cu_k, a.B, a.tk, base + at);
        behind = __builtin_amdgcn_readlane((int)(sq.start + sq.len - 1 - q), at);
        break;
      }
    }
  }
  const int n = chunks_of(sk.len, parts.C);
  if (n == 1) return;
  float top = -__FLT_MAX__;
  for (int i = lane; i < n; i += 64) top = fmaxf(top, parts.m[i * parts.n + p]);
  top = wave_max(top);
  float total = 0.f;
  for (int i = lane; i < n; i += 64) total += parts.l[i * parts.n + p] * exp2_hw(parts.m[i * parts.n + p] - top);
  total = wave_sum(total);
  const float inv = total != 0.f ? 1.f / total : nothing(a.causal ? sk.len - behind : sk.len);
  T* op = row_ptr<T>(a.o, batch, row, head);
  const int vecs = a.D / 4;
  if (lane < vecs) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < n; ++i) {
      const int64_t at = i * parts.n + p;
      const float f = parts.l[at] * exp2_hw(parts.m[at] - top) * inv;
      const f32x4 y = *reinterpret_cast<const f32x4*>(parts.o + at * a.D + 4 * lane);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += y[j] * f;
    }
    store4(op + 4 * lane, v[0], v[1], v[2], v[3]);
    if (a.low) store_low4<T>(a.low + p * a.D + 4 * lane, v[0], v[1], v[2], v[3]);
  }
  if (lane == 0 && a.lse) a.lse[p] = total == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(total)) * LN2;
}

template <class T, int DP, int NW>
static int launch_rows_dp(const Args& a, const Parts& parts, int most_chunks, hipStream_t s) {
  const int64_t slots = a.cu_k ? a.tk / parts.C + a.B + 2 : (int64_t)a.B * (a.tk > 0 ? (a.tk + parts.C - 1) / parts.C : 1);
  if (slots > 0x7fffffffLL || a.Hkv > 65535) return forge_set_error(FORGE_ERR_INVALID, "attention: too many chunks");
  attn_rows_kernel<T, DP, NW><<<dim3((unsigned)slots, a.Hkv), NW * 64, 0, s>>>(a, parts);
  FORGE_CHECK_LAUNCH();
  if (most_chunks > 1) {
    attn_join_kernel<T><<<(unsigned)((parts.n + 3) / 4), 256, 0, s>>>(a, parts);
    FORGE_CHECK_LAUNCH();
  }
  return FORGE_OK;
}

// Keys a chunk: about three workgroups a CU (one or two are resident at a time, and
// the lengths differ; two a CU took 120 us, four 118, three 117), at least 128 keys,
// and partial sums of at most 512 MB.
static int chunk_keys(const Args& a, int64_t n) {
  int64_t C = (a.cu_k ? a.tk : a.tk * a.B) * a.Hkv / 768;
  const int64_t most = (int64_t(512) << 20) / ((a.D + 2) * 4);  // (chunk, query, head)
  while (n * (a.tk / (C < 128 ? 128 : C) + 1) > most && C < a.tk) C = C < 128 ? 256 : 2 * C;
  C = (C + 127) / 128 * 128;
  return (int)(C < 128 ? 128 : C > (1 << 30) ? (1 << 30) : C);
}

int64_t rows_workspace(const Args& a, int64_t n_queries) {
  const int64_t n = n_queries * a.H;
  const int C = chunk_keys(a, n);
  if (a.tk <= C) return 0;
  return (a.tk / C + 1) * n * (a.D + 2) * 4;
}

int launch_rows(int dtype, const Args& a, int64_t n_queries, void* work, hipStream_t s) {
  Parts parts = {};
  parts.n = n_queries * a.H;
  if (parts.n == 0) return FORGE_OK;
  parts.C = chunk_keys(a, parts.n);
  const int64_t most = a.tk <= parts.C ? 1 : a.tk / parts.C + 1;
  if (most > 1) {
    if (!work || !aligned16(work)) return forge_set_error(FORGE_ERR_INVALID, "attention: work is NULL or not aligned");
    parts.o = (float*)work;
    parts.m = parts.o + most * parts.n * a.D;
    parts.l = parts.m + most * parts.n;
  }
  const int m = (int)(most > 1 ? 2 : 1);
  // (D 128: with 2 waves two workgroups are resident, one's beginning and end under
  // the other's stream: the 32 sequences above, with 4 waves 117 us, with 2 112)
  if (dtype == FORGE_DTYPE_F16) {
    if (a.D <= 64) return launch_rows_dp<fp16_t, 64, 4>(a, parts, m, s);
    if (a.D <= 128) return launch_rows_dp<fp16_t, 128, 2>(a, parts, m, s);
    return launch_rows_dp<fp16_t, 256, 2>(a, parts, m, s);
  }
  if (a.D <= 64) return launch_rows_dp<bf16_t, 64, 4>(a, parts, m, s);
  if (a.D <= 128) return launch_rows_dp<bf16_t, 128, 2>(a, parts, m, s);
  return launch_rows_dp<bf16_t, 256, 2>(a, parts, m, s);
}

}  // namespace fattn
