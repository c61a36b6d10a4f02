// RMS norm of every query and key head and its rotary embedding, in one pass
// over q and k, for gfx950; forward and backward.
//
// Per head x of D values, with r = 1 / sqrt(mean(x^2) + eps), n = x r,
// w = weight + offset and the half-split rotation R of the token's position:
//     out = R (n w)
// and, with dy = R^T dout (R is orthogonal: the same rotation by -theta),
//     dweight = sum over tokens and heads of dy n
//     g = dy w,   dx = r (g - n mean(g n)).
// Everything is fp32 between the loads and the one rounding of each output.
//
// Bound by HBM: forward 2 and backward 3 passes over q and k.  A head is
// shared by L lanes (a power of two): lane c owns 16 bytes at c of the lower
// half and the 16 bytes they rotate with in the upper half, so nothing leaves
// the lane but the sum of squares (and the mean of g n).  A lane takes two
// heads of a token together, which share the token's place, its row of the
// table and the loads in flight.  Measured on MI355X, bf16 [4, 4096], 32 + 8
// heads of 128, nothing cached: forward 63 us (5.3 TB/s; a copy 5.8), backward
// 92 us without and 102 us with the weights' gradients (5.5 and 4.9 TB/s).
//
// A head_dim whose half is no power of two of 16 bytes leaves lanes idle (96: 6 of
// 8, 4.2 TB/s both ways; 80: 5 of 8, 3.4), one whose half is no multiple of 16
// bytes (72: 2.1 TB/s), or a tensor off 16 bytes, takes 8 columns a lane at any
// alignment and the last lane's one by one (all of them one by one: 0.6).
//
// Weight gradients: a workgroup adds up its heads in registers and writes one
// row of partial sums, so there are few of them, each with the same share of
// the heads: 768 (3 per CU, what the registers of two heads allow) 102 us; 1024
// with one head a lane 106; 2048 110, 4096 119 (more rows to add up, and a last
// round that is not full).  The adds within a wave go by DPP: the step from
// ds_bpermute took the backward from 119 to 115 us, on a larger grid than this.
#include "common.h"

namespace {

constexpr int kBlock = 256;
constexpr int kMaxHalf = 512;      // head_dim up to 1024
constexpr int kMaxBlocks = 16384;  // 64 workgroups per CU
constexpr int kDwBlocks = 768;     // with weight gradients: 3 workgroups per CU, each one row of partial sums
constexpr int kHeads = 2;          // heads of a token that a lane takes together

// (batch, head, seq) element strides of a [B, heads, S, D] tensor
struct View {
  int64_t sb, sh, ss;
};

struct Side {  // q or k
  const void* x; View xv;
  const void* dy; View dv;   // backward: gradient of the output
  void* out; View ov;        // forward: the output; backward: dx
  const void* w;
  float* part;               // backward: [blocks][D] partial sums of dweight, or nullptr
  uint32_t tokens, heads;    // tokens = B * S
  uint32_t blocks;
};

struct Args {
  Side q, k;
  const void* cos; int64_t cos_sb, cos_ss;
  const void* sin; int64_t sin_sb, sin_ss;
  const int64_t* positions;
  int64_t table_rows;
  uint32_t seq_len;
  int half, lanes;
  float eps, offset, inv_d;
  int w_dtype;
};

// Sum over the L lanes that share a head, by DPP within 16 lanes: neighbours,
// pairs of a quad, then mirrored halves, whose lanes already agree.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

__device__ __forceinline__ float head_sum(float v, int lanes) {
  if (lanes >= 2) v = add_dpp<0xb1>(v);    // quad_perm [1, 0, 3, 2]
  if (lanes >= 4) v = add_dpp<0x4e>(v);    // quad_perm [2, 3, 0, 1]
  if (lanes >= 8) v = add_dpp<0x141>(v);   // row_half_mirror
  if (lanes >= 16) v = add_dpp<0x140>(v);  // row_mirror
  if (lanes >= 32) v += __shfl_xor(v, 16, 64);
  if (lanes >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// 16 bytes at an address that is a multiple of the element only (global memory
// takes them at any)
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// A lane's values of one half of a head: E columns at c * E.  VEC: 16 aligned
// bytes, and every lane's columns are there.  Otherwise (tensors off 16 bytes, or
// a half that is no multiple of 16 bytes) 8 columns, of which the last lane may
// have fewer.
template <class T, bool VEC>
struct Lane {
  static constexpr int E = VEC ? 16 / (int)sizeof(T) : 8;
  int c, half;
  __device__ __forceinline__ bool on(int j) const { return VEC || c * E + j < half; }
  __device__ __forceinline__ bool full() const { return VEC || c * E + E <= half; }

  // The values as they are in memory (cos and sin may be of another type TC).
  template <class S, bool NT>
  struct Raw {
    static constexpr int PER = 16 / (int)sizeof(S);
    Vec16<S> v[E < PER ? 1 : E / PER];
  };
  template <class S, bool NT>
  __device__ __forceinline__ void load(const S* p, Raw<S, NT>& r) const {
    constexpr int PER = Raw<S, NT>::PER;
    p += c * E;
    if constexpr (E < PER) {  // 16-bit weights of fp32 heads: less than 16 bytes
#pragma unroll
      for (int j = 0; j < E; ++j) r.v[0].v[j] = on(j) ? p[j] : from_f32<S>(0.f);
    } else if (full()) {
#pragma unroll
      for (int k = 0; k < E / PER; ++k) {
        if constexpr (VEC) {
          r.v[k] = NT ? load16_nt(p + k * PER) : load16(p + k * PER);
        } else {
          const u32x4_any w = *reinterpret_cast<const u32x4_any*>(p + k * PER);
          r.v[k].raw = make_uint4(w.x, w.y, w.z, w.w);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) r.v[j / PER].v[j % PER] = on(j) ? p[j] : from_f32<S>(0.f);
    }
  }
  template <class S, bool NT>
  __device__ __forceinline__ void values(const Raw<S, NT>& r, float (&v)[E]) const {
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = to_f32(r.v[j / Raw<S, NT>::PER].v[j % Raw<S, NT>::PER]);
  }
  template <class S>
  __device__ __forceinline__ void plus(const S* p, float offset, float (&v)[E]) const {
    Raw<S, false> r;
    load(p, r);
    values(r, v);
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] += offset;
  }
  __device__ __forceinline__ void weight(const void* w, int dtype, int first, float offset, float (&v)[E]) const {
    if (dtype == FORGE_DTYPE_BF16) plus((const bf16_t*)w + first, offset, v);
    else if (dtype == FORGE_DTYPE_F16) plus((const fp16_t*)w + first, offset, v);
    else plus((const float*)w + first, offset, v);
  }
  __device__ __forceinline__ void store(T* p, const float (&v)[E]) const {
    constexpr int PER = 16 / (int)sizeof(T);
    Vec16<T> t[E / PER];
#pragma unroll
    for (int j = 0; j < E; ++j) t[j / PER].v[j % PER] = from_f32<T>(v[j]);
    p += c * E;
    if (full()) {
#pragma unroll
      for (int k = 0; k < E / PER; ++k) {
        if constexpr (VEC) {
          store16_nt(p + k * PER, t[k]);
        } else {
          const u32x4_any w = {t[k].raw.x, t[k].raw.y, t[k].raw.z, t[k].raw.w};
          *reinterpret_cast<u32x4_any*>(p + k * PER) = w;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (on(j)) p[j] = t[j / PER].v[j % PER];
    }
  }
};

template <class T, class TC, bool VEC, bool SEQ, bool BWD, bool DW, bool LATE>
__global__ __launch_bounds__(kBlock) void qk_norm_rope_kernel(Args a) {
  using LaneT = Lane<T, VEC>;
  using X = typename LaneT::template Raw<T, true>;
  using C = typename LaneT::template Raw<TC, false>;
  constexpr int E = LaneT::E;
  constexpr int HEADS = kHeads;
  extern __shared__ float lds[];  // DW: [waves][D]
  const bool is_k = blockIdx.x >= a.q.blocks;
  const Side& s = is_k ? a.k : a.q;
  const uint32_t block = is_k ? blockIdx.x - a.q.blocks : blockIdx.x;
  const int lanes = a.lanes, half = a.half;
  const LaneT lane{(int)threadIdx.x & (lanes - 1), half};
  const bool active = lane.c * E < half;
  const uint32_t per_block = kBlock / lanes, step = s.blocks * per_block;
  const uint32_t groups = (s.heads + HEADS - 1) / HEADS, items = s.tokens * groups;

  float wl[E] = {}, wh[E] = {}, al[E], ah[E];  // weight of the lower and upper half, and their gradients' sums
  bool fresh = LATE;
  if (!LATE && active) {
    lane.weight(s.w, a.w_dtype, 0, a.offset, wl);
    lane.weight(s.w, a.w_dtype, half, a.offset, wh);
  }
#pragma unroll
  for (int j = 0; j < E; ++j) al[j] = ah[j] = 0.f;

  for (uint32_t item = block * per_block + threadIdx.x / lanes; item < items; item += step) {
    uint32_t b, sq, h0;
    if constexpr (SEQ) {
      const uint32_t r = item / a.seq_len;
      sq = item - r * a.seq_len;
      b = r / groups;
      h0 = (r - b * groups) * HEADS;
    } else {
      const uint32_t r = item / groups;
      h0 = (item - r * groups) * HEADS;
      b = r / a.seq_len;
      sq = r - b * a.seq_len;
    }
    X rl[HEADS] = {}, rh[HEADS] = {}, dl[HEADS] = {}, dh[HEADS] = {};
    C rc = {}, rs = {};
    const T* x = (const T*)s.x + ((int64_t)b * s.xv.sb + (int64_t)h0 * s.xv.sh + (int64_t)sq * s.xv.ss);
#pragma unroll
    for (int u = 0; u < HEADS; ++u)
      if (active && h0 + u < s.heads) {
        lane.load(x + u * s.xv.sh, rl[u]);
        lane.load(x + u * s.xv.sh + half, rh[u]);
      }
    if constexpr (BWD) {
      const T* dy = (const T*)s.dy + ((int64_t)b * s.dv.sb + (int64_t)h0 * s.dv.sh + (int64_t)sq * s.dv.ss);
#pragma unroll
      for (int u = 0; u < HEADS; ++u)
        if (active && h0 + u < s.heads) {
          lane.load(dy + u * s.dv.sh, dl[u]);
          lane.load(dy + u * s.dv.sh + half, dh[u]);
        }
    }
    const int64_t pos = a.positions ? a.positions[(int64_t)b * a.seq_len + sq] : (int64_t)sq;
    const bool in_table = pos >= 0 && pos < a.table_rows;
    if (active && in_table) {
      lane.load((const TC*)a.cos + ((int64_t)b * a.cos_sb + pos * a.cos_ss), rc);
      lane.load((const TC*)a.sin + ((int64_t)b * a.sin_sb + pos * a.sin_ss), rs);
    }
    if constexpr (LATE) {
      if (fresh && active) {
        lane.weight(s.w, a.w_dtype, 0, a.offset, wl);
        lane.weight(s.w, a.w_dtype, half, a.offset, wh);
      }
      fresh = false;
    }
    float cs[E], sn[E];
    lane.values(rc, cs);
    lane.values(rs, sn);
    T* o = (T*)s.out + ((int64_t)b * s.ov.sb + (int64_t)h0 * s.ov.sh + (int64_t)sq * s.ov.ss);
#pragma unroll
    for (int u = 0; u < HEADS; ++u) {
      float xl[E], xh[E];
      lane.values(rl[u], xl);
      lane.values(rh[u], xh);
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) ss += xl[j] * xl[j] + xh[j] * xh[j];
      float r = rsqrtf(head_sum(ss, lanes) * a.inv_d + a.eps);
      if (!in_table) r = __builtin_nanf("");  // nothing of the table was read: the token's outputs are NaN
      if (HEADS > 1 && h0 + u >= s.heads) r = 0.f;  // no head: x = dy = 0, which an eps of 0 would turn into NaN
      if constexpr (!BWD) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float yl = xl[j] * r * wl[j], yh = xh[j] * r * wh[j];
          xl[j] = yl * cs[j] - yh * sn[j];
          xh[j] = yh * cs[j] + yl * sn[j];
        }
      } else {
        float gl[E], gh[E];
        lane.values(dl[u], gl);
        lane.values(dh[u], gh);
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          // r dy; then r g = r dy w, and with sum g n = sum (r g) x
          const float yl = (gl[j] * cs[j] + gh[j] * sn[j]) * r, yh = (gh[j] * cs[j] - gl[j] * sn[j]) * r;
          if constexpr (DW) {  // (a head past the last one adds zeros)
            al[j] += yl * xl[j];
            ah[j] += yh * xh[j];
          }
          gl[j] = yl * wl[j];
          gh[j] = yh * wh[j];
          dot += gl[j] * xl[j] + gh[j] * xh[j];
        }
        // dx = r g - n r mean(g n)
        const float m = head_sum(dot, lanes) * a.inv_d * r * r;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          xl[j] = gl[j] - xl[j] * m;
          xh[j] = gh[j] - xh[j] * m;
        }
      }
      if (active && h0 + u < s.heads) {
        lane.store(o + u * s.ov.sh, xl);
        lane.store(o + u * s.ov.sh + half, xh);
      }
    }
  }

  if constexpr (DW) {
    if (!s.part) return;  // (uniform over the workgroup)
    // this workgroup's row of partial sums, in a fixed order: the groups of a
    // wave by shuffles, then the waves
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j < E; ++j)
      for (int off = lanes; off < 64; off <<= 1) {
        al[j] += __shfl_xor(al[j], off, 64);
        ah[j] += __shfl_xor(ah[j], off, 64);
      }
    if ((int)(threadIdx.x & 63) < lanes && active) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (lane.on(j)) {
          lds[wave * 2 * half + lane.c * E + j] = al[j];
          lds[wave * 2 * half + half + lane.c * E + j] = ah[j];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * half; i += kBlock) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kBlock / 64; ++w) v += lds[w * 2 * half + i];
      s.part[(int64_t)block * 2 * half + i] = v;
    }
  }
}

// dweight[i] = sum over the workgroups' partial sums, in a fixed order: 32
// columns a workgroup, 32 threads to a column.  blockIdx.y: q or k.
__global__ __launch_bounds__(1024) void qk_dweight_kernel(const float* qp, uint32_t q_blocks, void* dqw, const float* kp,
                                                          uint32_t k_blocks, void* dkw, int d, int w_dtype) {
  __shared__ float red[32][33];
  const float* part = blockIdx.y ? kp : qp;
  const int n = (int)(blockIdx.y ? k_blocks : q_blocks);
  void* out = blockIdx.y ? dkw : dqw;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + x;
  if (!part) return;  // (uniform)
  float v = 0.f;
  if (i < d) {
#pragma unroll 8
    for (int b = y; b < n; b += 32) v += part[(int64_t)b * d + i];
  }
  red[y][x] = v;
  __syncthreads();
  if (y == 0 && i < d) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += red[k][x];
    if (w_dtype == FORGE_DTYPE_BF16) ((bf16_t*)out)[i] = (bf16_t)t;
    else if (w_dtype == FORGE_DTYPE_F16) ((fp16_t*)out)[i] = (fp16_t)t;
    else ((float*)out)[i] = t;
  }
}

int lanes_for(int64_t half, int64_t each) {
  int lanes = 1;
  while (lanes * each < half) lanes <<= 1;
  return lanes;
}

// Workgroups of q and k: all they can use up to the cap, shared by their heads
// (at least one each: the cap is far above two).
void split_blocks(Args& a, int heads_each, uint64_t cap) {
  const uint64_t all = (uint64_t)a.q.heads + a.k.heads, per = kBlock / a.lanes;
  for (Side* s : {&a.q, &a.k}) {
    const uint64_t items = (uint64_t)s->tokens * ((s->heads + heads_each - 1) / heads_each);
    uint64_t most = all ? cap * s->heads / all : 0;
    if (most == 0) most = 1;
    const uint64_t b = (items + per - 1) / per;
    s->blocks = (uint32_t)(b > most ? most : b);
  }
}

// A call of few workgroups, a serving step's, is as long as its chain of loads:
// there the weights are asked for behind the first heads (bf16, 16 tokens, 32 + 8
// heads of 128: 4.5 us against 6.1), and so they are by the few workgroups that
// add up weight gradients.  Where many workgroups follow each other the order
// does not matter, and the test in the loop costs 3 us of 63 ([4, 4096]).
constexpr uint32_t kFewBlocks = 1024;

template <class T, class TC, bool VEC, bool SEQ, bool BWD>
void launch_as(const Args& a, uint32_t blocks, size_t lds, hipStream_t s) {
  if constexpr (BWD) {
    if (lds) qk_norm_rope_kernel<T, TC, VEC, SEQ, true, true, true><<<blocks, kBlock, lds, s>>>(a);
    else qk_norm_rope_kernel<T, TC, VEC, SEQ, true, false, false><<<blocks, kBlock, 0, s>>>(a);
  } else {
    if (blocks <= kFewBlocks) qk_norm_rope_kernel<T, TC, VEC, SEQ, false, false, true><<<blocks, kBlock, 0, s>>>(a);
    else qk_norm_rope_kernel<T, TC, VEC, SEQ, false, false, false><<<blocks, kBlock, 0, s>>>(a);
  }
}

template <class T, class TC, bool BWD>
void launch(const Args& a, bool vec, bool seq_first, uint32_t blocks, size_t lds, hipStream_t s) {
  if (!vec) launch_as<T, TC, false, false, BWD>(a, blocks, lds, s);
  else if (seq_first) launch_as<T, TC, true, true, BWD>(a, blocks, lds, s);
  else launch_as<T, TC, true, false, BWD>(a, blocks, lds, s);
}

template <bool BWD>
int run(int dtype, const char* what, Args& a, int w_dtype, int table_dtype, int64_t batch, int64_t n_q, int64_t n_kv,
        int64_t seq_len, int64_t head_dim, double eps, double offset, void* dqw, void* dkw, float* work, void* stream) {
  if (batch < 0 || n_q < 0 || n_kv < 0 || seq_len < 0)
    return forge_set_error(FORGE_ERR_INVALID, "%s: negative shape", what);
  if (head_dim <= 0 || head_dim % 2 != 0 || head_dim / 2 > kMaxHalf)
    return forge_set_error(FORGE_ERR_INVALID, "%s: head_dim %lld (even, up to %d)", what, (long long)head_dim, 2 * kMaxHalf);
  if (dtype != FORGE_DTYPE_F32 && dtype != FORGE_DTYPE_BF16 && dtype != FORGE_DTYPE_F16)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  if (w_dtype != FORGE_DTYPE_F32 && w_dtype != FORGE_DTYPE_BF16 && w_dtype != FORGE_DTYPE_F16)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: weight dtype %d", what, w_dtype);
  if (table_dtype != dtype && table_dtype != FORGE_DTYPE_F32)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: cos/sin dtype %d with q dtype %d (tables are q's dtype or fp32)",
                           what, table_dtype, dtype);
  if (a.table_rows < 0) return forge_set_error(FORGE_ERR_INVALID, "%s: negative table_rows", what);
  if (!a.positions && a.table_rows < seq_len)
    return forge_set_error(FORGE_ERR_INVALID, "%s: cos/sin have %lld rows for seq_len %lld", what,
                           (long long)a.table_rows, (long long)seq_len);
  const int64_t lim = 0x40000000;  // rows, and a grid's step past them, stay below 2^32
  if (batch > lim || n_q > lim || n_kv > lim || seq_len > lim || batch * seq_len > lim ||
      batch * seq_len * (n_q > n_kv ? n_q : n_kv) > lim)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "%s: more than 2^30 heads in a call", what);
  const int64_t tokens = batch * seq_len;
  for (const Side* s : {&a.q, &a.k})
    if (tokens * (s == &a.q ? n_q : n_kv) > 0 && (!s->x || !s->out || !s->w || (BWD && !s->dy)))
      return forge_set_error(FORGE_ERR_INVALID, "%s: an array of q or k is NULL", what);
  if (tokens * (n_q + n_kv) > 0 && (!a.cos || !a.sin))
    return forge_set_error(FORGE_ERR_INVALID, "%s: cos or sin is NULL", what);
  if ((dqw || dkw) && !work) return forge_set_error(FORGE_ERR_INVALID, "%s: weight gradients need the workspace", what);

  const size_t es = dtype_size(dtype), ets = dtype_size(table_dtype);
  const int64_t V = (int64_t)(16 / es), Vt = (int64_t)(16 / ets);
  a.half = (int)(head_dim / 2);
  bool vec = a.half % V == 0 && a.half / V <= 64 && aligned16(a.cos) && aligned16(a.sin) && aligned16(a.q.w) &&
             aligned16(a.k.w);
  for (const Side* s : {&a.q, &a.k}) {
    vec = vec && aligned16(s->x) && aligned16(s->out) && (!BWD || aligned16(s->dy));
    for (int64_t st : {s->xv.sb, s->xv.sh, s->xv.ss, s->ov.sb, s->ov.sh, s->ov.ss}) vec = vec && st % V == 0;
    if (BWD)
      for (int64_t st : {s->dv.sb, s->dv.sh, s->dv.ss}) vec = vec && st % V == 0;
  }
  for (int64_t st : {a.cos_sb, a.cos_ss, a.sin_sb, a.sin_ss}) vec = vec && st % Vt == 0;
  a.lanes = lanes_for(a.half, vec ? V : 8);
  a.seq_len = (uint32_t)seq_len;
  a.eps = (float)eps;
  a.offset = (float)offset;
  a.inv_d = (float)(1.0 / (double)head_dim);
  a.w_dtype = w_dtype;
  a.q.heads = (uint32_t)n_q;
  a.k.heads = (uint32_t)n_kv;
  // a wave's heads lie next to each other in memory: heads of a token in [B, S,
  // H, D] memory, tokens of a head in [B, H, S, D] (bf16 [4, 32 + 8, 7324, 128],
  // forward / backward: by tokens 105 / 176 us, by heads 128 / 202)
  const bool seq_first = n_q > 1 && seq_len > 1 && a.q.xv.ss < a.q.xv.sh;
  a.q.tokens = a.k.tokens = (uint32_t)(batch * seq_len);
  hipStream_t s = (hipStream_t)stream;
  const bool dw = dqw || dkw;
  split_blocks(a, kHeads, dw ? kDwBlocks : kMaxBlocks);
  if (dw) {  // both sides' partial sums, one after the other
    a.q.part = dqw ? work : nullptr;
    a.k.part = dkw ? work + (int64_t)a.q.blocks * head_dim : nullptr;
  }
  const uint32_t blocks = a.q.blocks + a.k.blocks;
  if (blocks) {
    const size_t lds = dw ? (kBlock / 64) * (size_t)head_dim * sizeof(float) : 0;
    const bool f32_table = table_dtype != dtype;
    switch (dtype) {
      case FORGE_DTYPE_F32: launch<float, float, BWD>(a, vec, seq_first, blocks, lds, s); break;
      case FORGE_DTYPE_BF16:
        if (f32_table) launch<bf16_t, float, BWD>(a, vec, seq_first, blocks, lds, s);
        else launch<bf16_t, bf16_t, BWD>(a, vec, seq_first, blocks, lds, s);
        break;
      default:
        if (f32_table) launch<fp16_t, float, BWD>(a, vec, seq_first, blocks, lds, s);
        else launch<fp16_t, fp16_t, BWD>(a, vec, seq_first, blocks, lds, s);
    }
    FORGE_CHECK_LAUNCH();
  }
  if (dw) {  // (no rows: zeros)
    qk_dweight_kernel<<<dim3((unsigned)((head_dim + 31) / 32), 2), 1024, 0, s>>>(
        a.q.part, a.q.blocks, dqw, a.k.part, a.k.blocks, dkw, (int)head_dim, w_dtype);
    FORGE_CHECK_LAUNCH();
  }
  return FORGE_OK;
}

}  // namespace

extern "C" int forge_qk_norm_rope_fwd(int dtype, const void* q, int64_t q_sb, int64_t q_sh, int64_t q_ss, const void* k,
                                      int64_t k_sb, int64_t k_sh, int64_t k_ss, void* q_out, int64_t qo_sb,
                                      int64_t qo_sh, int64_t qo_ss, void* k_out, int64_t ko_sb, int64_t ko_sh,
                                      int64_t ko_ss, const void* q_weight, const void* k_weight, int w_dtype,
                                      const void* cos, int64_t cos_sb, int64_t cos_ss, const void* sin, int64_t sin_sb,
                                      int64_t sin_ss, int table_dtype, int64_t table_rows, const int64_t* positions,
                                      int64_t batch, int64_t n_q, int64_t n_kv, int64_t seq_len, int64_t head_dim,
                                      double eps, double offset, void* stream) {
  Args a = {};
  a.q = {q, {q_sb, q_sh, q_ss}, nullptr, {}, q_out, {qo_sb, qo_sh, qo_ss}, q_weight, nullptr, 0, 0, 0};
  a.k = {k, {k_sb, k_sh, k_ss}, nullptr, {}, k_out, {ko_sb, ko_sh, ko_ss}, k_weight, nullptr, 0, 0, 0};
  a.cos = cos; a.cos_sb = cos_sb; a.cos_ss = cos_ss;
  a.sin = sin; a.sin_sb = sin_sb; a.sin_ss = sin_ss;
  a.positions = positions;
  a.table_rows = table_rows;
  return run<false>(dtype, "qk_norm_rope_fwd", a, w_dtype, table_dtype, batch, n_q, n_kv, seq_len, head_dim, eps, offset,
                    nullptr, nullptr, nullptr, stream);
}

extern "C" int64_t forge_qk_norm_rope_bwd_workspace(int64_t head_dim) {
  return (kDwBlocks + 2) * head_dim * (int64_t)sizeof(float);
}

extern "C" int forge_qk_norm_rope_bwd(int dtype, const void* dq, int64_t dq_sb, int64_t dq_sh, int64_t dq_ss,
                                      const void* dk, int64_t dk_sb, int64_t dk_sh, int64_t dk_ss, const void* q,
                                      int64_t q_sb, int64_t q_sh, int64_t q_ss, const void* k, int64_t k_sb,
                                      int64_t k_sh, int64_t k_ss, void* dq_in, int64_t qi_sb, int64_t qi_sh,
                                      int64_t qi_ss, void* dk_in, int64_t ki_sb, int64_t ki_sh, int64_t ki_ss,
                                      const void* q_weight, const void* k_weight, int w_dtype, const void* cos,
                                      int64_t cos_sb, int64_t cos_ss, const void* sin, int64_t sin_sb, int64_t sin_ss,
                                      int table_dtype, int64_t table_rows, const int64_t* positions, void* dq_weight,
                                      void* dk_weight, void* work, int64_t batch, int64_t n_q, int64_t n_kv,
                                      int64_t seq_len, int64_t head_dim, double eps, double offset, void* stream) {
  Args a = {};
  a.q = {q, {q_sb, q_sh, q_ss}, dq, {dq_sb, dq_sh, dq_ss}, dq_in, {qi_sb, qi_sh, qi_ss}, q_weight, nullptr, 0, 0, 0};
  a.k = {k, {k_sb, k_sh, k_ss}, dk, {dk_sb, dk_sh, dk_ss}, dk_in, {ki_sb, ki_sh, ki_ss}, k_weight, nullptr, 0, 0, 0};
  a.cos = cos; a.cos_sb = cos_sb; a.cos_ss = cos_ss;
  a.sin = sin; a.sin_sb = sin_sb; a.sin_ss = sin_ss;
  a.positions = positions;
  a.table_rows = table_rows;
  return run<true>(dtype, "qk_norm_rope_bwd", a, w_dtype, table_dtype, batch, n_q, n_kv, seq_len, head_dim, eps, offset,
                   dq_weight, dk_weight, (float*)work, stream);
}
