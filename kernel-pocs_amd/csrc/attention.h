// What the attention kernels share: arguments, the sequences of a packed
// batch and their tiles, LDS tiles of keys or queries, and the fragments that
// v_mfma_f32_32x32x16 takes from them.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i),  s_ij = scale q_i . k_j,
// over the keys j that query i sees: all of its sequence's, or (causal) j <= i +
// len_k - len_q, so that the last query sees every key.  A query that sees
// none has o = 0 and lse = -inf; one whose scores are all -inf has o = NaN, as softmax.
//
// Sequences: cu_q and cu_k hold the B + 1 offsets of each, or are NULL for B
// dense sequences of len_q and len_k rows.  Row i of sequence s lies at base +
// s * batch stride + i * row stride (varlen: batch stride 0, i from the start
// of the array).  Rows before the first offset and behind the last are
// sequences -1 and B without a counterpart on the other side: their outputs and
// gradients are zeros.  Offsets are clamped to the array and to their
// predecessor, so wrong ones give wrong results, never an access outside it.
#pragma once

#include <type_traits>

#include "gemm_core.h"

namespace fattn {

using fgemm::bf16x8;
using fgemm::f32x16;
using fgemm::f32x4;
using fgemm::make_rsrc;
using fgemm::mfma16;
using fgemm::mfma32;
using fgemm::OOB;
using fgemm::tr_frag;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int NXCD = 8;

struct Rows {  // [batch][row][head][D] with unit stride in D
  const void* p;
  int64_t batch, row, head;
};

struct Args {
  Rows q, k, v, o, dout, dq, dk, dv;  // o: an output of the forward, an input of the backward
  float* lse;                         // [queries][H] natural logarithms
  int8_t* low;                        // [queries][H][D], what the rounding of o left, or NULL
  float* delta;                       // [queries][H], sum of o dout (backward)
  const int32_t* cu_q;
  const int32_t* cu_k;
  int B;
  int64_t tq, tk;                     // rows of the arrays (varlen), or of one sequence (dense)
  int H, Hkv, D;
  float scale;
  int causal;
  float* part;                        // dk and dv of `parts` parts of a group's heads, [part][row][Hkv][2][D]
  int parts;                          // 1: dk and dv are written as they are
};

// The forward's p = exp2(s c - m), m the running maximum of s c less P_UP.  fp16's
// smallest step is 2^-24: with p up to 1 the keys more than 17 below a maximum (in
// natural units) counted for nothing in o, however many they are, and in full in l.
// Held 2^9 times as large, as far as the maximum's steps of 2^6 let it, p has them to 2^-34.
template <class T>
constexpr float P_UP = std::is_same_v<T, fp16_t> ? 9.f : 0.f;

template <class T> __device__ __forceinline__ T* row_ptr(const Rows& r, int64_t batch, int64_t row, int head) {
  return (T*)r.p + batch * r.batch + row * r.row + head * r.head;
}

// A sequence on one side: rows [start, start + len) of batch entry `batch`.
struct Span {
  int64_t batch, start;
  int len;
};

__device__ __forceinline__ Span span_of(const int32_t* cu, int B, int64_t total, int s) {
  if (!cu) return {s, 0, s >= 0 && s < B ? (int)total : 0};
  const int64_t a = s < 0 ? 0 : min(max((int64_t)cu[s], (int64_t)0), total);
  int64_t b = s >= B ? total : min(max((int64_t)cu[s + 1], a), total);
  return {0, a, (int)(b - a)};
}

// Tiles of `rows` rows of the sequences on one side, in order of the sequences
// -1 .. B: the sequence of tile t and its index there (seq > B: no such tile).
// A wave looks at 64 sequences at once.
struct TileAt {
  int seq, tile;
};

// least: tiles that a sequence without rows counts as.
__device__ __forceinline__ TileAt find_tile(const int32_t* cu, int B, int64_t total, int rows, int t, int least = 0) {
  if (!cu) {
    const int per = max((int)((total + rows - 1) / rows), least);
    if (per == 0 || t >= per * B) return {B + 1, 0};
    return {t / per, t % per};
  }
  const int lane = threadIdx.x % 64;
  for (int base = -1; base <= B; base += 64) {
    const int s = base + lane;
    int n = 0;
    if (s <= B) n = max((span_of(cu, B, total, s).len + rows - 1) / rows, least);
    int sum = n;  // inclusive prefix sum
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const int up = __shfl_up(sum, off, 64);
      if (lane >= off) sum += up;
    }
    const uint64_t past = __ballot(sum > t);
    if (past) {
      const int at = __builtin_ctzll(past);
      return {base + at, t - __builtin_amdgcn_readlane(sum - n, at)};
    }
    t -= __builtin_amdgcn_readlane(sum, 63);
  }
  return {B + 1, 0};
}

// The same tiles in the order of `level`, the number of the tile from its
// sequence's other end: the first tile of n has level n for the keys, the last
// one for the queries, so that (causal) the tiles with the most work come first
// and the last workgroups to start are short ones (13 sequences of 70 to 420
// tokens, 14 heads of 64 on 2: the dk, dv kernel 113 -> 90 us).  More than 254
// sequences go in their own order: there are many tiles then, and short ones.
struct LevelAt {
  int seq, level;  // level: 1 .. tiles of the sequence
};

__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return __builtin_amdgcn_readfirstlane(v);
}

// (What follows from it is the same in all lanes, and has to be seen as that: a
// sequence's length in vector registers drove the dk, dv kernel's others to
// scratch memory.)
__device__ __forceinline__ LevelAt find_level(const int32_t* cu, int B, int64_t total, int rows, int t) {
  if (!cu) {
    const int per = (int)((total + rows - 1) / rows);
    if (per == 0 || t >= per * B) return {B + 1, 1};
    return {t % B, per - t / B};
  }
  if (B > 254) {
    const TileAt at = find_tile(cu, B, total, rows, t);
    if (at.seq > B) return {B + 1, 1};
    return {at.seq, (span_of(cu, B, total, at.seq).len + rows - 1) / rows - at.tile};
  }
  const int lane = threadIdx.x % 64;
  int n[4], top = 0;  // tiles of sequences -1 + 64 c + lane
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int s = -1 + 64 * c + lane;
    n[c] = s <= B ? (span_of(cu, B, total, s).len + rows - 1) / rows : 0;
    top = max(top, n[c]);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = max(top, __shfl_xor(top, off, 64));
  top = __builtin_amdgcn_readfirstlane(top);
  auto from = [&](int level) {  // tiles of this level and above
    int sum = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) sum += max(0, n[c] - level + 1);
    return wave_sum_int(sum);
  };
  if (from(1) <= t) return {B + 1, 1};
  int lo = 1, hi = top;  // the largest level with more than t tiles from it on
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (from(mid) > t) lo = mid;
    else hi = mid - 1;
  }
  int left = t - from(lo + 1);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint64_t has = __ballot(n[c] >= lo);
    const int count = __builtin_popcountll(has);
    if (left < count) {
      const bool mine = (has >> lane & 1) && __builtin_popcountll(has & ((uint64_t(1) << lane) - 1)) == left;
      return {-1 + 64 * c + (int)__builtin_ctzll(__ballot(mine)), lo};
    }
    left -= count;
  }
  return {B + 1, 1};
}

// At most this many tiles of `rows` rows (host).
inline int64_t most_tiles(const int32_t* cu, int B, int64_t total, int rows) {
  if (!cu) return (int64_t)B * ((total + rows - 1) / rows);
  return total / rows + B + 2;
}

// ---------------------------------------------------------------------------
// LDS tiles: rows of DP 16-bit values (DP = 64, 128 or 256) in units of 4 rows (8
// of 128 bytes), 16 bytes between units; in a unit the 16-byte chunks of a row
// are exchanged by an XOR with f(row).  A fragment is read either by rows (32
// rows, one chunk each: 16 neighbouring rows must lie in different chunks of the
// 256-byte bank cycle) or transposed (four rows, 64 bytes each: those must lie in
// different quarters of it).  Both hold: f exchanges the quarters among the rows of a
// unit, and the gaps shift the units by a chunk each.  As f changes few bits of a
// chunk's number and nothing beyond a unit, most of a read's address is an
// immediate: four bases a lane serve all reads of one kind (an XOR of all four
// bits, without gaps, took 16, and the dk, dv kernel kept them in scratch memory).
// ---------------------------------------------------------------------------
template <int DP>
struct Tile {
  static constexpr int RB = DP * 2, CPR = RB / 16;  // bytes and chunks of a row
  static constexpr int UNIT = DP == 64 ? 8 : 4;     // rows of a unit
  static constexpr int UB = UNIT * RB + 16;         // bytes from unit to unit
  static constexpr int bytes(int rows) { return rows / UNIT * UB; }
  static __device__ __forceinline__ int f(int row) {
    if constexpr (DP == 64) return 4 * ((row >> 1) & 1) + 2 * ((row >> 2) & 1);
    else return 4 * (row & 3);
  }
};

// One LDS-DMA instruction: 16 (4) bytes of each lane, from its offset to lds +
// 16 (4) lane.  (The host's pass over this code does not know the 16-byte form.)
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t off, int scalar_off) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, off, scalar_off, 0, 0);
#endif
}
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t off) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 4, off, 0, 0, 0);
#endif
}

// LDS-DMA of ROWS rows by NW waves: an instruction fills 1 KB (half a unit at DP = 256).
template <int DP, int ROWS, int NW>
struct TileDma {
  typedef Tile<DP> L;
  static constexpr int RPI = 64 / L::CPR, N = ROWS / RPI / NW;  // rows of an instruction, instructions of a wave
  static_assert(ROWS % (RPI * NW) == 0 && N >= 1 && (DP < 256 || N % 2 == 0), "whole instructions and units");
  static constexpr int BYTES = L::bytes(ROWS);
  int step;             // bytes of RPI rows
  uint32_t off[DP == 256 ? 2 : 1];  // this lane's chunk from the instruction's first row (OOB: past D), by parity

  __device__ __forceinline__ void setup(int64_t row_stride, int D) {
    const int lane = threadIdx.x % 64;
    step = (int)(row_stride * 2) * RPI;
#pragma unroll
    for (int p = 0; p < (DP == 256 ? 2 : 1); ++p) {
      const int row = p * RPI + lane / L::CPR, chunk = (lane % L::CPR) ^ L::f(row);
      off[p] = chunk * 8 < D ? (uint32_t)(lane / L::CPR * (int)(row_stride * 2) + chunk * 16) : OOB;
    }
  }
  // rows from `left` on do not exist and read as zeros, as do columns from D on
  __device__ __forceinline__ void load(const void* first, int left, char* dst, int wave) const {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(first);
    const int lane_row = threadIdx.x % 64 / L::CPR;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = wave * N + j;
      char* to = dst + (DP == 256 ? i / 2 * L::UB + i % 2 * 1024 : i * L::UB);
      const uint32_t o = off[DP == 256 ? j % 2 : 0];
      dma16(r, to, i * RPI + lane_row < left ? o : OOB, i * step);
    }
  }
};

// Fragments by rows: rows r0 .. r0 + 31 (r0 a multiple of 32), columns 16 ks .. + 15:
// lane l holds row l % 32, columns 16 ks + 8 (l / 32) .. + 7.
template <int DP>
struct RowFrag {
  typedef Tile<DP> L;
  int base[4];  // of the chunks whose bits that f changes are those of 0 .. 3
  __device__ __forceinline__ void setup(int lane) {
    const int row = lane % 32, h = lane / 32;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      base[i] = row / L::UNIT * L::UB + row % L::UNIT * L::RB + ((((DP == 64 ? 2 : 4) * i + h) ^ L::f(row)) << 4);
  }
  __device__ __forceinline__ bf16x8 read(const char* tile, int r0, int ks) const {
    const int at = r0 / L::UNIT * L::UB + (DP == 64 ? 0 : ks % 2 * 32 + ks / 8 * 256);
    return *reinterpret_cast<const bf16x8*>(tile + base[DP == 64 ? ks : ks / 2 % 4] + at);
  }
};

// Fragments of the transposed tile: columns 32 db .. + 31 (lane l holds column 32 db
// + l % 32), rows r0 + 4 h + {0 .. 3} and r0 + 8 + 4 h + {0 .. 3}, h = l / 32, r0 a
// multiple of 16: the rows in the order in which an accumulator of 32 x 32
// holds them, so that its registers 8 i .. 8 i + 7, rounded, are the other operand.
template <int DP>
struct ColFrag {
  typedef Tile<DP> L;
  static constexpr int NB = DP == 64 ? 2 : 4;
  int base[NB];
  __device__ __forceinline__ void setup(int lane) {
    const int q = 4 * (lane / 32) + lane % 16 / 4, c = 16 * (lane / 16 % 2) + 4 * (lane % 4);
#pragma unroll
    for (int i = 0; i < NB; ++i)
      base[i] = q / L::UNIT * L::UB + q % L::UNIT * L::RB + (((4 * i + c / 8) ^ L::f(q)) << 4) + c % 8 * 2;
  }
  __device__ __forceinline__ bf16x8 read(const char* tile, int r0, int db) const {
    const char* p = tile + base[db % NB] + r0 / L::UNIT * L::UB + db / NB * 256;
    return tr_frag(p, p + 8 / L::UNIT * L::UB);
  }
};

// Keys that a query does not see have p = 0, but 0 times an infinity or NaN is NaN,
// and a product takes 16 keys at once.  Kernels run as if there were none; where
// a causal sum comes out as NaN or infinite they run again with such values apart: added
// to the sums of the queries that see them, and zeros in the tile.  (Seldom runs: few
// registers, not speed.  No value of a finite tile passes through any of this.)  For the
// keys' gradients it is 16 queries at once, and they know beforehand.
template <class T, int DP>
struct Special {
  typedef Tile<DP> L;
  static constexpr uint32_t EX = std::is_same_v<T, fp16_t> ? 0x7c00 : 0x7f80;
  static __device__ __forceinline__ char* row_at(char* tile, int row) { return tile + row / L::UNIT * L::UB + row % L::UNIT * L::RB; }
  static __device__ __forceinline__ bool is(uint32_t half) { return (half & EX) == EX; }

  static __device__ __forceinline__ bool in_row(char* tile, int row) {
    bool any = false;
    for (int w = threadIdx.x % 64; w < DP / 2; w += 64) {
      const uint32_t x = reinterpret_cast<const uint32_t*>(row_at(tile, row))[w];
      any |= is(x) || is(x >> 16);
    }
    return __any(any);
  }
  // those of rows r0 .. r0 + n - 1 whose number, first + j, is from `lo` on and below `hi`;
  // as they are (times a p above 0) or as NaN
  static __device__ __forceinline__ void add(f32x16 (&sums)[DP / 32], char* tile, int r0, int n, int first, int lo, int hi, bool as_nan) {
    const int h = threadIdx.x % 64 / 32;
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const int row = r0 + j;
      if (!in_row(tile, row)) continue;
      const char* p = row_at(tile, row);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (r % 4 == 0) __builtin_amdgcn_sched_barrier(0);
          const int d = 32 * db + 8 * (r / 4) + 4 * h + r % 4;
          const uint16_t x = *reinterpret_cast<const uint16_t*>(p + ((d / 8 ^ L::f(row)) << 4) + d % 8 * 2);
          const float v = as_nan ? __builtin_nanf("") : to_f32(__builtin_bit_cast(T, x));
          sums[db][r] += is(x) && first + j >= lo && first + j < hi ? v : 0.f;
        }
    }
  }
  // zeros in their places, and the others times `by`, a power of two (not in fp16); by
  // waves `wave` of `waves`
  static __device__ __forceinline__ void clear(char* tile, int r0, int n, int wave, int waves, float by = 1.f) {
#pragma unroll 1
    for (int row = r0 + wave; row < r0 + n; row += waves)
      for (int w = threadIdx.x % 64; w < DP / 2; w += 64) {
        uint32_t* p = reinterpret_cast<uint32_t*>(row_at(tile, row)) + w;
        uint32_t x = *p;
        if (!is(x) && !is(x >> 16) && by == 1.f) continue;
        x = (is(x) ? 0 : x & 0xffff) | (is(x >> 16) ? 0 : x & 0xffff0000u);
        if (by != 1.f)
          x = __float_as_uint(__uint_as_float(x << 16) * by) >> 16 | (__float_as_uint(__uint_as_float(x & 0xffff0000u) * by) & 0xffff0000u);
        *p = x;
      }
  }
};

// The second run's factor of the values, a power of two, for n keys: sums of p below 2^6
// times values near bf16's largest pass fp32's range, and the result, divided by the sum
// of p, does not.  With it they do not either, and no other bit changes but of values
// below 2^-87.  (fp16's values are far from that.)
template <class T>
__device__ __forceinline__ float v_down(int n) {
  n = __builtin_amdgcn_readfirstlane(n);  // (the same in all lanes, and held once)
  return std::is_same_v<T, fp16_t> ? 1.f : __uint_as_float((uint32_t)(127 - 7 - (32 - __builtin_clz(n | 1))) << 23);
}
// 1 / l of a query that has no probability: of one that sees no key 0, and so are its sums;
// of one whose keys' scores are all -inf NaN, which its softmax is.
__device__ __forceinline__ float nothing(int sees) { return sees > 0 ? __builtin_nanf("") : 0.f; }

// whether a first run with values that are not finite is to be followed by a second
template <class T>
__device__ __forceinline__ bool second_run(bool hides) { return hides || !std::is_same_v<T, fp16_t>; }

// (infinities among them; in four chains)
template <int N>
__device__ __forceinline__ bool any_nan(const f32x16 (&sums)[N]) {
  float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) t[r % 4] = __builtin_fmaf(sums[i][r], 0.f, t[r % 4]);
  const float all = t[0] + t[1] + (t[2] + t[3]);
  return all != all;
}

// Whether any of the workgroup's 4 waves has it; through 16 bytes of LDS that no wave
// reads any more after the first barrier.  (__syncthreads_or has an array of its own,
// beside which the compiler no longer tells the tiles that are read from those
// under way: it waited for the LDS-DMA before each tile's first read, 396 -> 430 us
// for 329 GFLOP.)
__device__ __forceinline__ bool any_of_4_waves(char* lds, int wave, bool has) {
  const bool mine = __any(has);
  __syncthreads();
  if (threadIdx.x % 64 == 0) reinterpret_cast<int*>(lds)[wave] = mine;
  __syncthreads();
  const int4 v = *reinterpret_cast<const int4*>(lds);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(v.x | v.y | v.z | v.w) != 0;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// two values rounded to 16 bits (nearest even), in one word
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef T t2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), t2));
}

// registers 8 i .. 8 i + 7 of an accumulator as an operand
template <class T>
__device__ __forceinline__ bf16x8 pack_acc(const f32x16& a, int i) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = pack2<T>(a[8 * i + 2 * j], a[8 * i + 2 * j + 1]);
  return __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
}

// four values rounded and stored
template <class T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(a, b), pack2<T>(c, d));
}

// What rounding x took, in 254ths of a step of the rounded value r: delta = sum o dout
// is formed of r + low.  (Of r alone it misses by roundings of o, and every ds of the
// row then has that error: some 15% more in dq and dk, for a byte a value.)
template <class T>
__device__ __forceinline__ float low_step(float r) {
  const float e = __uint_as_float(__float_as_uint(r) & 0x7f800000u);
  return std::is_same_v<T, fp16_t> ? fmaxf(e, 0x1p-14f) * (0x1p-10f / 254.f) : fmaxf(e, 0x1p-100f) * (0x1p-7f / 254.f);
}
template <class T>
__device__ __forceinline__ uint32_t low_byte(float x) {
  const float r = to_f32(from_f32<T>(x));
  return (uint32_t)(int)rintf(fminf(fmaxf((x - r) / low_step<T>(r), -127.f), 127.f)) & 255u;
}
template <class T>
__device__ __forceinline__ void store_low4(int8_t* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint32_t*>(p) = low_byte<T>(a) | low_byte<T>(b) << 8 | low_byte<T>(c) << 16 | low_byte<T>(d) << 24;
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// this wave's LDS-DMA has landed, but for the last N instructions, and its LDS reads are done
template <int N> __device__ __forceinline__ void wait_dma() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
  asm volatile("" ::: "memory");
}

// bare workgroup barrier: LDS accesses do not move across it, and LDS-DMA in
// flight is not waited for (each wave waits for its own before it)
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Which (tile, head) a workgroup takes.  Workgroups go to the XCDs in turn;
// the heads of a group share keys and values, so an XCD takes whole groups (or
// a part of the tiles of one, where there are fewer groups than XCDs) and its
// L2 holds them once.
struct Item {
  int tile, kv, g;  // g: head within the group, or 0
};
__device__ __forceinline__ Item item_of(int id, int tiles, int Hkv, int G) {
  if (Hkv % NXCD == 0) {
    const int x = id % NXCD, i = id / NXCD;
    return {i / G % tiles, x + NXCD * (i / G / tiles), i % G};
  }
  if (NXCD % Hkv == 0) {
    const int share = NXCD / Hkv, x = id % NXCD, i = id / NXCD;
    return {(i / G) * share + x / Hkv, x % Hkv, i % G};
  }
  return {id / G / Hkv, id / G % Hkv, id % G};
}
inline int64_t items(int64_t tiles, int Hkv, int G) {
  if (Hkv % NXCD == 0 || NXCD % Hkv != 0) return tiles * Hkv * G;
  const int share = NXCD / Hkv;
  return (tiles + share - 1) / share * NXCD * G;
}

}  // namespace fattn
