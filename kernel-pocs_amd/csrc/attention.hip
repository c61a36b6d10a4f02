// Entry points of attention: argument checks and the choice of the kernel.
#include "attention.h"

namespace fattn {

int launch_fwd(int dtype, const Args& a, hipStream_t s);
int launch_rows(int dtype, const Args& a, int64_t n_queries, void* work, hipStream_t s);
int64_t rows_workspace(const Args& a, int64_t n_queries);
int launch_bwd(int dtype, const Args& a, float* shift, int64_t n_rows, hipStream_t s);
int dkv_parts(const Args& a);

// Few queries a sequence: the kernel that reads keys by chunks.  The lengths are
// on the device, so the rule goes by their mean: at most 4 queries a sequence
// whose heads' rows fill one tile of 32.
static bool few_queries(const Args& a, int64_t n_queries) {
  return n_queries <= 4 * (int64_t)a.B && n_queries * (a.H / a.Hkv) <= 32 * (int64_t)a.B;
}

static int check_rows(const char* name, const Rows& r, int64_t n_batch, int64_t n_rows, int64_t n_heads) {
  if (n_rows == 0 || n_heads == 0 || n_batch == 0) return FORGE_OK;
  if (!r.p) return forge_set_error(FORGE_ERR_INVALID, "attention: %s is NULL", name);
  if (!aligned16(r.p) || r.batch % 8 || r.row % 8 || r.head % 8)
    return forge_set_error(FORGE_ERR_INVALID, "attention: %s needs 16-byte aligned rows", name);
  // a tile's offsets are 32-bit bytes from its first row
  if (r.row < 0 || r.head < 0 || r.batch < 0 || r.row >= (int64_t(1) << 23))
    return forge_set_error(FORGE_ERR_INVALID, "attention: %s row stride %lld", name, (long long)r.row);
  return FORGE_OK;
}

static int check_sizes(int dtype, const Args& a) {
  if (dtype != FORGE_DTYPE_F16 && dtype != FORGE_DTYPE_BF16)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "attention: dtype %d", dtype);
  if (a.B < 0 || a.tq < 0 || a.tk < 0 || a.tq > 0x7fffffff || a.tk > 0x7fffffff)
    return forge_set_error(FORGE_ERR_INVALID, "attention: sizes");
  if (a.D < 8 || a.D > 256 || a.D % 8)
    return forge_set_error(FORGE_ERR_UNSUPPORTED, "attention: head_dim %d (a multiple of 8 up to 256)", a.D);
  if (a.H < 1 || a.Hkv < 1 || a.H % a.Hkv)
    return forge_set_error(FORGE_ERR_INVALID, "attention: %d heads on %d key heads", a.H, a.Hkv);
  if ((a.cu_q == nullptr) != (a.cu_k == nullptr))
    return forge_set_error(FORGE_ERR_INVALID, "attention: offsets of one side only");
  // (the backward divides lse by it, and all multiply it by log2(e))
  if (!(a.scale >= 0x1p-100f && a.scale <= 0x1p100f)) return forge_set_error(FORGE_ERR_INVALID, "attention: scale %g", a.scale);
  return FORGE_OK;
}

static Args make_args(const int32_t* cu_q, const int32_t* cu_k, int64_t B, int64_t tq, int64_t tk, int64_t H, int64_t Hkv,
                      int64_t D, float scale, int causal) {
  Args a = {};
  auto narrow = [](int64_t v) { return v < 0 ? -1 : v > 0x7ffffff0 ? -1 : (int)v; };
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.B = narrow(B);
  a.tq = tq;
  a.tk = tk;
  a.H = narrow(H);
  a.Hkv = narrow(Hkv);
  a.D = narrow(D);
  a.scale = scale;
  a.causal = causal != 0;
  return a;
}

}  // namespace fattn

using namespace fattn;

extern "C" int64_t forge_attention_fwd_workspace(int varlen, int64_t B, int64_t tq, int64_t tk, int64_t H, int64_t Hkv,
                                                 int64_t D) {
  static const int32_t none = 0;
  const int32_t* cu = varlen ? &none : nullptr;  // (only whether it is NULL is looked at)
  const Args a = make_args(cu, cu, B, tq, tk, H, Hkv, D, 1.f, 1);
  if (check_sizes(FORGE_DTYPE_BF16, a)) return -1;
  const int64_t n = varlen ? tq : B * tq;
  return n > 0 && few_queries(a, n) ? rows_workspace(a, n) : 0;
}

extern "C" int forge_attention_fwd(int dtype, const void* q, int64_t q_batch, int64_t q_row, int64_t q_head,
                                   const void* k, int64_t k_batch, int64_t k_row, int64_t k_head,
                                   const void* v, int64_t v_batch, int64_t v_row, int64_t v_head,
                                   void* out, int64_t o_batch, int64_t o_row, int64_t o_head, float* lse, int8_t* low,
                                   const int32_t* cu_q, const int32_t* cu_k, int64_t B, int64_t tq, int64_t tk,
                                   int64_t H, int64_t Hkv, int64_t D, float scale, int causal, void* work, void* stream) {
  Args a = make_args(cu_q, cu_k, B, tq, tk, H, Hkv, D, scale, causal);
  if (int e = check_sizes(dtype, a)) return e;
  a.q = {q, q_batch, q_row, q_head};
  a.k = {k, k_batch, k_row, k_head};
  a.v = {v, v_batch, v_row, v_head};
  a.o = {out, o_batch, o_row, o_head};
  a.lse = lse;
  a.low = low;
  if (!aligned16(low)) return forge_set_error(FORGE_ERR_INVALID, "attention: low is not 16-byte aligned");
  const int64_t nb = cu_q ? 1 : B, n = nb * tq;
  if (int e = check_rows("q", a.q, nb, tq, H)) return e;
  if (int e = check_rows("k", a.k, nb, tk, Hkv)) return e;
  if (int e = check_rows("v", a.v, nb, tk, Hkv)) return e;
  if (int e = check_rows("out", a.o, nb, tq, H)) return e;
  if (n == 0) return FORGE_OK;
  if (few_queries(a, n)) return launch_rows(dtype, a, n, work, (hipStream_t)stream);
  return launch_fwd(dtype, a, (hipStream_t)stream);
}

// -delta and -lse / scale by head and query, and dk and dv of parts of a group's heads
static int64_t stat_bytes(int64_t n_queries, int64_t H) { return (n_queries * H * 2 * 4 + 15) / 16 * 16; }

extern "C" int64_t forge_attention_bwd_workspace(int varlen, int64_t B, int64_t tq, int64_t tk, int64_t H, int64_t Hkv,
                                                 int64_t D) {
  static const int32_t none = 0;
  const int32_t* cu = varlen ? &none : nullptr;  // (only whether it is NULL is looked at)
  const Args a = make_args(cu, cu, B, tq, tk, H, Hkv, D, 1.f, 1);
  if (check_sizes(FORGE_DTYPE_BF16, a)) return -1;
  const int parts = dkv_parts(a);
  return stat_bytes(varlen ? tq : B * tq, H) + (parts > 1 ? (int64_t)parts * (varlen ? tk : B * tk) * Hkv * 2 * D * 4 : 0);
}

extern "C" int forge_attention_bwd(int dtype, const void* dout, int64_t do_batch, int64_t do_row, int64_t do_head,
                                   const void* q, int64_t q_batch, int64_t q_row, int64_t q_head,
                                   const void* k, int64_t k_batch, int64_t k_row, int64_t k_head,
                                   const void* v, int64_t v_batch, int64_t v_row, int64_t v_head,
                                   const void* out, int64_t o_batch, int64_t o_row, int64_t o_head, const float* lse,
                                   const int8_t* low, void* dq, int64_t dq_batch, int64_t dq_row, int64_t dq_head,
                                   void* dk, int64_t dk_batch, int64_t dk_row, int64_t dk_head,
                                   void* dv, int64_t dv_batch, int64_t dv_row, int64_t dv_head,
                                   const int32_t* cu_q, const int32_t* cu_k, int64_t B, int64_t tq, int64_t tk,
                                   int64_t H, int64_t Hkv, int64_t D, float scale, int causal, void* work, void* stream) {
  Args a = make_args(cu_q, cu_k, B, tq, tk, H, Hkv, D, scale, causal);
  if (int e = check_sizes(dtype, a)) return e;
  a.q = {q, q_batch, q_row, q_head};
  a.k = {k, k_batch, k_row, k_head};
  a.v = {v, v_batch, v_row, v_head};
  a.o = {out, o_batch, o_row, o_head};
  a.dout = {dout, do_batch, do_row, do_head};
  a.dq = {dq, dq_batch, dq_row, dq_head};
  a.dk = {dk, dk_batch, dk_row, dk_head};
  a.dv = {dv, dv_batch, dv_row, dv_head};
  a.lse = const_cast<float*>(lse);
  a.low = const_cast<int8_t*>(low);
  const int64_t nb = cu_q ? 1 : B, n = nb * tq;
  if (int e = check_rows("dout", a.dout, nb, tq, H)) return e;
  if (int e = check_rows("q", a.q, nb, tq, H)) return e;
  if (int e = check_rows("k", a.k, nb, tk, Hkv)) return e;
  if (int e = check_rows("v", a.v, nb, tk, Hkv)) return e;
  if (int e = check_rows("out", a.o, nb, tq, H)) return e;
  if (int e = check_rows("dq", a.dq, nb, tq, H)) return e;
  if (int e = check_rows("dk", a.dk, nb, tk, Hkv)) return e;
  if (int e = check_rows("dv", a.dv, nb, tk, Hkv)) return e;
  if (n > 0 && (!lse || !low || !work)) return forge_set_error(FORGE_ERR_INVALID, "attention: lse, low or work is NULL");
  if (!aligned16(work) || !aligned16(low)) return forge_set_error(FORGE_ERR_INVALID, "attention: work or low is not aligned");
  a.delta = (float*)work;
  a.parts = n > 0 ? dkv_parts(a) : 1;
  a.part = (float*)((char*)work + stat_bytes(n, H));
  return launch_bwd(dtype, a, (float*)work + n * H, n, (hipStream_t)stream);
}
