// What the attention kernels share: arguments, the sequences of a packed
// batch and their tiles, LDS tiles of keys or queries, and the fragments that
// v_mfma_f32_32x32x16 takes from them.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i),  s_ij = scale q_i . k_j,
// over the keys j that query i sees: all of its sequence's, or (causal) j <= i +
// len_k - len_q, so that the last query sees every key.  A query that sees
// none has o = 0 and lse = -inf.
//
// Sequences: cu_q and cu_k hold the B + 1 offsets of each, or are NULL for B
// dense sequences of len_q and len_k rows.  Row i of sequence s lies at base +
// s * batch stride + i * row stride (varlen: batch stride 0, i from the start
// of the array).  Rows before the first offset and behind the last are
// sequences -1 and B without a counterpart on the other side: their outputs and
// gradients are zeros.  Offsets are clamped to the array and to their
// predecessor, so wrong ones give wrong results, never an access outside it.
#pragma once

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
  float* delta;                       // [queries][H], sum of o dout (backward)
  const int32_t* cu_q;
  const int32_t* cu_k;
  int B;
  int64_t tq, tk;                     // rows of the arrays (varlen), or of one sequence (dense)
  int H, Hkv, D;
  float scale;
  int causal;
};

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
      const int before = __shfl(sum - n, at, 64);
      return {__builtin_amdgcn_readfirstlane(base + at), __builtin_amdgcn_readfirstlane(t - before)};
    }
    t -= __shfl(sum, 63, 64);
  }
  return {B + 1, 0};
}

// At most this many tiles of `rows` rows (host).
inline int64_t most_tiles(const int32_t* cu, int B, int64_t total, int rows) {
  if (!cu) return (int64_t)B * ((total + rows - 1) / rows);
  return total / rows + B + 2;
}

// ---------------------------------------------------------------------------
// LDS tiles: rows of DP 16-bit values (DP = 64, 128 or 256), unpadded, the
// 16-byte chunks of a row exchanged by an XOR with a function of the row.  A
// fragment is read either by rows (32 rows, one chunk each: 16 neighbouring
// rows must lie in different chunks of the 256-byte bank cycle) or transposed
// (four rows, 64 bytes each: those must lie in different quarters of it).
// Both hold for
//   256- and 512-byte rows: 4 (row % 4) + row / 4 % 4
//   128-byte rows (two in a bank cycle): 4 (row / 2 % 2) + row / 4 % 4.
// ---------------------------------------------------------------------------
template <int DP>
__device__ __forceinline__ int swz_rows(int row) {
  if constexpr (DP == 64) return 4 * ((row >> 1) & 1) + ((row >> 2) & 3);
  else return 4 * (row & 3) + ((row >> 2) & 3);
}

// One LDS-DMA instruction: 16 (4) bytes of each lane, from its offset to lds +
// 16 (4) lane.  (The host's pass over this code does not know the 16-byte form.)
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t off) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, off, 0, 0, 0);
#endif
}
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t off) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 4, off, 0, 0, 0);
#endif
}

// LDS-DMA of ROWS rows by NW waves: instruction j of wave w fills 1 KB.
template <int DP, int ROWS, int NW>
struct TileDma {
  static constexpr int RB = DP * 2, CPR = RB / 16, RPI = 64 / CPR, N = ROWS / RPI / NW;
  static_assert(ROWS % (RPI * NW) == 0 && N >= 1, "whole instructions");
  static constexpr int BYTES = ROWS * RB;
  uint32_t off[N];  // byte offset of this lane's chunk from the tile's first row (OOB: past D)
  int row[N];       // its row

  __device__ __forceinline__ void setup(int64_t row_stride, int D, int wave) {
    const int lane = threadIdx.x % 64;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      row[j] = (wave * N + j) * RPI + lane / CPR;
      const int chunk = (lane % CPR) ^ swz_rows<DP>(row[j]);
      off[j] = chunk * 8 < D ? (uint32_t)(row[j] * (int)(row_stride * 2) + chunk * 16) : OOB;
    }
  }
  // rows from `left` on do not exist and read as zeros
  __device__ __forceinline__ void load(const void* first, int left, char* dst, int wave) const {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(first);
#pragma unroll
    for (int j = 0; j < N; ++j)
      dma16(r, dst + (wave * N + j) * 1024, row[j] < left ? off[j] : OOB);
  }
};

// Fragment by rows: rows r0 .. r0 + 31 (r0 a multiple of 32), columns 16 ks .. + 15:
// lane l holds row l % 32, columns 16 ks + 8 (l / 32) .. + 7.
template <int DP>
__device__ __forceinline__ bf16x8 frag_rows(const char* tile, int r0, int ks, int lane) {
  const int row = r0 + lane % 32;
  return *reinterpret_cast<const bf16x8*>(tile + row * (DP * 2) + (((2 * ks + lane / 32) ^ swz_rows<DP>(lane % 32)) << 4));
}

// Fragment of the transposed tile: columns c0 .. c0 + 31 (lane l holds column c0
// + l % 32), rows r0 + 4 h + {0 .. 3} and r0 + 8 + 4 h + {0 .. 3}, h = l / 32, r0 a
// multiple of 16: the rows in the order in which an accumulator of 32 x 32
// holds them, so that its registers 8 i .. 8 i + 7, rounded, are the other operand.
template <int DP>
struct TrOff {
  int lo, hi;  // byte offsets of the two reads at r0 = c0 = 0
  __device__ __forceinline__ void setup(int lane) {
    const int h = lane / 32, q = 4 * h + (lane % 16) / 4, c = 16 * ((lane / 16) % 2) + 4 * (lane % 4);
    lo = q * (DP * 2) + (((c / 8) ^ swz_rows<DP>(q)) << 4) + (c % 8) * 2;
    const int q8 = q + 8;
    hi = q8 * (DP * 2) + (((c / 8) ^ swz_rows<DP>(q8)) << 4) + (c % 8) * 2;
  }
};
// columns 32 db: chunks 4 db, an XOR of bits 6 and up of the offset with the row's swizzle in place
template <int DP>
__device__ __forceinline__ bf16x8 frag_cols(const char* tile, const TrOff<DP>& t, int r0, int db) {
  const char* p = tile + r0 * (DP * 2);
  return tr_frag(p + (t.lo ^ (db << 6)), p + (t.hi ^ (db << 6)));
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// registers 8 i .. 8 i + 7 of an accumulator as an operand
template <class T>
__device__ __forceinline__ bf16x8 pack_acc(const f32x16& a, int i) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const T lo = (T)a[8 * i + 2 * j], hi = (T)a[8 * i + 2 * j + 1];
    w[j] = (uint32_t)__builtin_bit_cast(uint16_t, lo) | ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16);
  }
  return __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
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
