"""RMS norm of every query and key head and RoPE, in one pass over q and k.

Models with q/k norms (Qwen3) norm each head between the projections
and the rotation: `q_norm`, `k_norm`, then `apply_rotary_pos_emb`
(forge/forge/patching/kernels/lora.py:254-264 of the reference runs them as
separate modules).  `apply_qk_norm_rope` does both at once, forward and
backward, with fp32 between the loads and one rounding of each output
(csrc/qk_norm_rope.hip); the separate modules round after the norm, after the
weight and in the rotation.

Layouts are `apply_rope`'s: q [B, n_q, S, D] and k [B, n_kv, S, D] with any
(batch, head, seq) strides, so HF's `transpose(1, 2)` views, or slices of one
packed projection, are read in place; outputs have the inputs' memory order.
n_q and n_kv are independent, D is even and at most 1024.  A call under
`torch.no_grad()` (a serving step: S = 1, `positions` [B, 1]) is one launch.
"""
from __future__ import annotations

from typing import Optional

import torch

from forge_hip import _lib as L
from .forge_rope_v3 import _tables, _unit_last

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_INTEGERS = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)
MAX_HEAD_DIM = 1024


def _check(q, k, q_weight, k_weight, cos, sin, positions, eps):
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"q and k must be [batch, heads, seq, head_dim], got {tuple(q.shape)} and {tuple(k.shape)}")
    B, _, S, D = q.shape
    kb, _, ks, kd = k.shape
    if kb != B or ks != S or kd != D:
        raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)} in batch, seq or head_dim")
    if D == 0 or D % 2 or D > MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be even and at most {MAX_HEAD_DIM}, got {D}")
    dtype, w_dtype = q.dtype, q_weight.dtype
    if dtype not in _DTYPES or w_dtype not in _DTYPES:
        raise TypeError(f"q, k and the weights must be fp16, bf16 or fp32, got {dtype} and {w_dtype}")
    if k.dtype != dtype:
        raise TypeError(f"q and k must have the same dtype, got {dtype} and {k.dtype}")
    if q_weight.shape != (D,) or k_weight.shape != (D,):
        raise ValueError(f"q_weight and k_weight must be [{D}], got {tuple(q_weight.shape)} and {tuple(k_weight.shape)}")
    if k_weight.dtype != w_dtype:
        raise TypeError(f"q_weight and k_weight must have the same dtype, got {w_dtype} and {k_weight.dtype}")
    if cos.dim() != 3 or cos.shape != sin.shape or cos.shape[0] not in (1, B) or cos.shape[2] != D:
        raise ValueError(f"cos and sin must be [1 or {B}, rows, {D}], got {tuple(cos.shape)} and {tuple(sin.shape)}")
    if not cos.is_floating_point() or not sin.is_floating_point():
        raise TypeError(f"cos and sin must be floating point, got {cos.dtype} and {sin.dtype}")
    if positions is None:
        if cos.shape[1] != S:
            raise ValueError(f"cos and sin have {cos.shape[1]} rows for {S} tokens; pass positions to index a table")
    else:
        if positions.dtype not in _INTEGERS:
            raise TypeError(f"positions must be an integer tensor (got {positions.dtype})")
        if positions.numel() != B * S:
            raise ValueError(f"positions must have batch * seq = {B * S} entries, got {positions.numel()}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    device = q.device
    if (k.device != device or q_weight.device != device or k_weight.device != device or cos.device != device
            or sin.device != device or (positions is not None and positions.device != device)):
        raise ValueError(f"every tensor must be on q's device {device}")
    L.require_gpu(q)


def _out_like(t):
    """An output in t's memory order, with a unit stride in head_dim."""
    out = torch.empty_like(t)
    return out if out.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _bhs(t):
    return t.stride()[:3]


def _table_strides(cos, sin, batch):
    """(batch, row) strides of each table; a table of one batch row serves all."""
    (cb, cs, _), (sb, ss, _) = cos.stride(), sin.stride()
    if cos.shape[0] != batch or batch == 1:
        cb = sb = 0
    return (cb, cs), (sb, ss)


def _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, offset):
    B, n_q, S, D = q.shape
    q_out, k_out = _out_like(q), _out_like(k)
    cos_st, sin_st = _table_strides(cos, sin, B)
    with L.on_device(q):
        L.check(
            L.forge_qk_norm_rope_fwd(
                L.dtype_code(q.dtype), q.data_ptr(), *_bhs(q), k.data_ptr(), *_bhs(k), q_out.data_ptr(), *_bhs(q_out),
                k_out.data_ptr(), *_bhs(k_out), q_weight.data_ptr(), k_weight.data_ptr(), L.dtype_code(q_weight.dtype),
                cos.data_ptr(), *cos_st, sin.data_ptr(), *sin_st, L.dtype_code(cos.dtype), cos.shape[1],
                L.ptr(positions), B, n_q, k.shape[1], S, D, eps, offset, L.stream_of(q)),
            "forge_qk_norm_rope_fwd")
    return q_out, k_out


def _backward(dq, dk, q, k, q_weight, k_weight, cos, sin, positions, eps, offset, need_qw, need_kw):
    B, n_q, S, D = q.shape
    dq, dk = _unit_last(dq), _unit_last(dk)
    dq_in, dk_in = _out_like(q), _out_like(k)
    dqw = torch.empty_like(q_weight) if need_qw else None
    dkw = torch.empty_like(k_weight) if need_kw else None
    work = None
    if need_qw or need_kw:
        work = torch.empty(L.forge_qk_norm_rope_bwd_workspace(D), device=q.device, dtype=torch.uint8)
    cos_st, sin_st = _table_strides(cos, sin, B)
    with L.on_device(q):
        L.check(
            L.forge_qk_norm_rope_bwd(
                L.dtype_code(q.dtype), dq.data_ptr(), *_bhs(dq), dk.data_ptr(), *_bhs(dk), q.data_ptr(), *_bhs(q),
                k.data_ptr(), *_bhs(k), dq_in.data_ptr(), *_bhs(dq_in), dk_in.data_ptr(), *_bhs(dk_in),
                q_weight.data_ptr(), k_weight.data_ptr(), L.dtype_code(q_weight.dtype), cos.data_ptr(), *cos_st,
                sin.data_ptr(), *sin_st, L.dtype_code(cos.dtype), cos.shape[1], L.ptr(positions), L.ptr(dqw), L.ptr(dkw),
                L.ptr(work), B, n_q, k.shape[1], S, D, eps, offset, L.stream_of(q)),
            "forge_qk_norm_rope_bwd")
    return dq_in, dk_in, dqw, dkw


class ForgeQKNormRoPEFunction(torch.autograd.Function):
    """forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps,
    offset) on arguments that `apply_qk_norm_rope` has checked and laid out;
    saves them, and the backward computes each head's norm again."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, offset):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps, ctx.offset = eps, offset
        return _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, offset)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        grads = _backward(dq, dk, *ctx.saved_tensors, ctx.eps, ctx.offset, *ctx.needs_input_grad[2:4])
        return (*grads, None, None, None, None, None)


def apply_qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                       cos: torch.Tensor, sin: torch.Tensor, positions: Optional[torch.Tensor] = None,
                       eps: float = 1e-6, offset: float = 0.0, validate_positions: bool = False):
    """(rope(rmsnorm(q) * (q_weight + offset)), the same of k).

    cos/sin [1 or B, rows, D] in q's dtype or fp32 (another dtype is widened
    to fp32), of which the first D/2 columns are read; rows == S, or
    `positions` (integers, B*S of them) gives each token's row.  A token whose
    position is outside the table reads nothing of it and comes out as NaN;
    validate_positions=True raises IndexError instead (one host sync).
    offset: 1.0 where the stored weight is the difference from one (Gemma).
    Gradients: q, k, and the weights where they require it."""
    _check(q, k, q_weight, k_weight, cos, sin, positions, eps)
    if positions is not None:
        if validate_positions and positions.numel():
            lo, hi = (int(v) for v in torch.aminmax(positions))
            if lo < 0 or hi >= cos.shape[1]:
                raise IndexError(f"positions must lie in [0, {cos.shape[1]}) (the cos/sin rows); got min {lo}, max {hi}")
        if positions.dtype != torch.int64 or not positions.is_contiguous():
            positions = positions.to(torch.int64).contiguous()
    cos, sin = _tables(cos, sin, q)
    q, k, q_weight, k_weight = _unit_last(q), _unit_last(k), q_weight.contiguous(), k_weight.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad
                                    or k_weight.requires_grad):
        return ForgeQKNormRoPEFunction.apply(q, k, q_weight, k_weight, cos, sin, positions, float(eps), float(offset))
    L.refuse_tangents(q, k, q_weight, k_weight, cos, sin)
    return _forward(q, k, q_weight, k_weight, cos, sin, positions, float(eps), float(offset))


class ForgeQKNormRoPE(torch.nn.Module):
    """The q and k norm weights of one attention layer, applied with RoPE."""

    def __init__(self, head_dim, eps=1e-6, offset=0.0, dtype=None, device=None):
        super().__init__()
        self.eps, self.offset = float(eps), float(offset)
        init = torch.zeros if self.offset == 1.0 else torch.ones
        self.q_weight = torch.nn.Parameter(init(head_dim, dtype=dtype, device=device))
        self.k_weight = torch.nn.Parameter(init(head_dim, dtype=dtype, device=device))

    def forward(self, q, k, cos, sin, positions=None):
        return apply_qk_norm_rope(q, k, self.q_weight, self.k_weight, cos, sin, positions, self.eps, self.offset)


__all__ = ["apply_qk_norm_rope", "ForgeQKNormRoPE", "ForgeQKNormRoPEFunction"]
