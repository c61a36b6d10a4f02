"""Attention with grouped heads, over packed sequences of different lengths or a
dense batch (csrc/attention_fwd.hip, attention_rows.hip, attention_bwd.hip).

    out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j - lse_i)

over the keys that query i sees: all of its sequence's or, causal, those j <= i +
len_k - len_q (the last query sees every key: a prompt, a prompt that continues
earlier tokens, or one token against a sequence's keys).  A query that sees no
key (a sequence without keys, or more queries than keys) has out = 0, lse = -inf
and no gradient.  One that sees keys whose scores are all -inf has no softmax: out and
the gradients that it takes part in are NaN, lse is -inf.

fp16 and bf16, head_dim a multiple of 8 up to 256, any number of heads on a
divisor of it.  Products take 16-bit operands (the probabilities and, backward,
their gradients are rounded to them) and sum in fp32; each result is rounded
once.  Every sum has a fixed order, forward and backward.  A key or value that is
not finite stays with the queries that see it, and a query, or a gradient that comes
in, with the keys that it sees.  Queries, keys and values are read where they lie
(columns of one projection's output, HF's transposed views); rows that are not 16-byte
aligned are copied first.
"""
from __future__ import annotations

from typing import Optional

import torch

from forge_hip import _lib as L

_DTYPES = (torch.float16, torch.bfloat16)
_INTEGERS = (torch.int32, torch.int64)
MAX_HEAD_DIM = 256
_MAX_ROW = 1 << 23  # elements from one token to the next
_SCALES = (2.0 ** -100, 2.0 ** 100)  # lse / scale and scale log2(e) within fp32


def _rows_ok(t, strides):
    batch, row, head = strides
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and row < _MAX_ROW and (batch | row | head) % 8 == 0


class _Layout:
    """(batch, row, head) strides of [T, heads, D] or [B, heads, S, D] tensors."""

    @staticmethod
    def packed(t):
        return (0, t.stride(0), t.stride(1))

    @staticmethod
    def dense(t):
        return (t.stride(0), t.stride(2), t.stride(1))


def _readable(t, layout):
    if _rows_ok(t, layout(t)):
        return t
    if layout is _Layout.packed:
        t = t.clone(memory_format=torch.contiguous_format)
    else:
        t = t.transpose(1, 2).clone(memory_format=torch.contiguous_format).transpose(1, 2)
    return t


def _new(shape, like, layout):
    """An output: tokens of all heads beside each other."""
    if layout is _Layout.packed:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    b, h, s, d = shape
    return torch.empty(b, s, h, d, dtype=like.dtype, device=like.device).transpose(1, 2)


def _sizes(q, k, cu_q, layout):
    """(batch, queries, keys, heads, key heads, head_dim) as the kernels take them."""
    if layout is _Layout.packed:
        return cu_q.numel() - 1, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2]
    return q.shape[0], q.shape[2], k.shape[2], q.shape[1], k.shape[1], q.shape[3]


def _forward(q, k, v, cu_q, cu_k, scale, causal, layout, want_lse, train=False):
    sizes = _sizes(q, k, cu_q, layout)
    out = _new(q.shape, q, layout)
    varlen = layout is _Layout.packed
    lse = low = None
    if train:  # what out's rounding took, for the gradients
        low = torch.empty(out.numel(), dtype=torch.int8, device=q.device)
    if want_lse:
        lse = torch.empty((q.shape[0], q.shape[1]) if varlen else (q.shape[0], q.shape[2], q.shape[1]),
                          dtype=torch.float32, device=q.device)
    if out.numel():
        nbytes = L.forge_attention_fwd_workspace(varlen, *sizes)
        work = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes > 0 else None
        with L.on_device(q):
            L.check(
                L.forge_attention_fwd(
                    L.dtype_code(q.dtype), q.data_ptr(), *layout(q), k.data_ptr(), *layout(k), v.data_ptr(), *layout(v),
                    out.data_ptr(), *layout(out), L.ptr(lse), L.ptr(low), L.ptr(cu_q), L.ptr(cu_k), *sizes,
                    scale, causal, L.ptr(work), L.stream_of(q)),
                "forge_attention_fwd")
    return out, lse, low


def _backward(dout, q, k, v, out, lse, low, cu_q, cu_k, scale, causal, layout):
    dout = _readable(dout, layout)
    sizes = _sizes(q, k, cu_q, layout)
    dq, dk, dv = _new(q.shape, q, layout), _new(k.shape, k, layout), _new(v.shape, v, layout)
    varlen = layout is _Layout.packed
    if q.numel() == 0:
        return dq, dk.zero_(), dv.zero_()
    work = torch.empty(L.forge_attention_bwd_workspace(varlen, *sizes), dtype=torch.uint8, device=q.device)
    with L.on_device(q):
        L.check(
            L.forge_attention_bwd(
                L.dtype_code(q.dtype), dout.data_ptr(), *layout(dout), q.data_ptr(), *layout(q), k.data_ptr(), *layout(k),
                v.data_ptr(), *layout(v), out.data_ptr(), *layout(out), lse.data_ptr(), L.ptr(low), dq.data_ptr(), *layout(dq),
                dk.data_ptr(), *layout(dk), dv.data_ptr(), *layout(dv), L.ptr(cu_q), L.ptr(cu_k), *sizes, scale, causal,
                work.data_ptr(), L.stream_of(q)),
            "forge_attention_bwd")
    return dq, dk, dv


class ForgeAttentionFunction(torch.autograd.Function):
    """forward(ctx, q, k, v, cu_q, cu_k, scale, causal, packed) -> (out, lse) on
    arguments that the entry points have checked and laid out; saves them with
    out, lse and a byte a value of what out's rounding took, and the backward computes
    the probabilities again."""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale, causal, packed):
        layout = _Layout.packed if packed else _Layout.dense
        out, lse, low = _forward(q, k, v, cu_q, cu_k, scale, causal, layout, True, True)
        ctx.save_for_backward(q, k, v, out, lse, low, cu_q, cu_k)
        ctx.args = (scale, causal, layout)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        dq, dk, dv = _backward(dout, *ctx.saved_tensors, *ctx.args)
        return dq, dk, dv, None, None, None, None, None


def _check(q, k, v, dims, scale):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != dims:
            raise ValueError(f"{name} must have {dims} dimensions, got {tuple(t.shape)}")
        if t.dtype not in _DTYPES:
            raise TypeError(f"q, k and v must be fp16 or bf16, got {t.dtype}")
        if t.dtype != q.dtype:
            raise TypeError(f"q, k and v must have the same dtype, got {q.dtype} and {t.dtype}")
        if t.device != q.device:
            raise ValueError(f"every tensor must be on q's device {q.device}")
    if k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have the same shape")
    D = q.shape[-1]
    if k.shape[-1] != D:
        raise ValueError(f"k's head_dim {k.shape[-1]} does not match q's {D}")
    if D < 8 or D % 8 or D > MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 8 up to {MAX_HEAD_DIM}, got {D}")
    heads, kv_heads = q.shape[1], k.shape[1]
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} heads need a number of key heads that divides them, got {kv_heads}")
    if scale is not None and not _SCALES[0] <= scale <= _SCALES[1]:
        raise ValueError(f"scale must be positive, from 2^-100 to 2^100, got {scale}")


def _offsets(name, cu, rows, device, validate):
    if cu.dim() != 1 or cu.numel() < 1 or cu.dtype not in _INTEGERS:
        raise ValueError(f"{name} must be a vector of int32 or int64 offsets, got {cu.dtype} {tuple(cu.shape)}")
    if cu.device != device:
        raise ValueError(f"every tensor must be on q's device {device}")
    if validate:
        at = cu.tolist()
        if at[0] != 0 or at[-1] > rows or any(a > b for a, b in zip(at, at[1:])):
            raise ValueError(f"{name} must begin at 0, not decrease and end at {rows} or before, got {at}")
    if cu.dtype != torch.int32:
        cu = cu.clamp(0, rows).to(torch.int32)
    return cu.contiguous()


def _apply(q, k, v, cu_q, cu_k, scale, causal, layout, return_lse):
    L.require_gpu(q)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    q, k, v = _readable(q, layout), _readable(k, layout), _readable(v, layout)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = ForgeAttentionFunction.apply(q, k, v, cu_q, cu_k, scale, bool(causal), layout is _Layout.packed)
    else:
        L.refuse_tangents(q, k, v)
        out, lse, _ = _forward(q, k, v, cu_q, cu_k, scale, bool(causal), layout, return_lse)
    return (out, lse) if return_lse else out


def forge_varlen_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                           cu_seqlens_k: Optional[torch.Tensor] = None, *, causal: bool = True,
                           scale: Optional[float] = None, return_lse: bool = False, validate_offsets: bool = False):
    """Attention of sequences packed without padding: q [T, heads, D], k and v [T_k,
    kv_heads, D] -> [T, heads, D] (and lse [T, heads] in fp32 with return_lse).

    Sequence i has the queries cu_seqlens[i] .. cu_seqlens[i + 1] - 1 and the keys
    that cu_seqlens_k gives in the same way (None: the queries' own).  Offsets begin
    at 0 and do not decrease; they are not read on the host, so the call can be
    captured and replayed with other lengths of the same totals.  Offsets that
    break this give wrong results but touch nothing outside the tensors;
    validate_offsets=True raises ValueError instead (a host sync).  Rows behind
    the last sequence come out as zeros and get zero gradients.  scale: default
    D ** -0.5.  Gradients: q, k, v; not through lse."""
    _check(q, k, v, 3, scale)
    cu_q = _offsets("cu_seqlens", cu_seqlens, q.shape[0], q.device, validate_offsets)
    if cu_seqlens_k is None:
        if k.shape[0] != q.shape[0]:
            raise ValueError(f"{k.shape[0]} keys for {q.shape[0]} queries need cu_seqlens_k")
        cu_k = cu_q
    else:
        cu_k = _offsets("cu_seqlens_k", cu_seqlens_k, k.shape[0], q.device, validate_offsets)
        if cu_k.numel() != cu_q.numel():
            raise ValueError(f"cu_seqlens has {cu_q.numel() - 1} sequences, cu_seqlens_k {cu_k.numel() - 1}")
    return _apply(q, k, v, cu_q, cu_k, scale, causal, _Layout.packed, return_lse)


def forge_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True,
                    scale: Optional[float] = None, return_lse: bool = False):
    """Attention of a dense batch: q [B, heads, S, D], k and v [B, kv_heads, S_k, D] in any
    strides -> [B, heads, S, D] in [B, S, heads, D] memory (and lse [B, S, heads] in
    fp32 with return_lse); otherwise as forge_varlen_attention."""
    _check(q, k, v, 4, scale)
    if k.shape[0] != q.shape[0]:
        raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)} in batch")
    return _apply(q, k, v, None, None, scale, causal, _Layout.dense, return_lse)


__all__ = ["ForgeAttentionFunction", "forge_attention", "forge_varlen_attention"]
