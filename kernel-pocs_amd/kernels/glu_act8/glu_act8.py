"""Gated activation act(gate) * up whose backward reads gate and up from an
8-bit copy (csrc/glu_act8.hip).

`swiglu` / `geglu` save gate and up as they are: 4 bytes a position in bf16,
the largest part of what a layer of a gated MLP holds between its passes.
`glu_act8` saves 2.06: groups of 32 values along a row share a power of two
2^e, the least with |x| <= 127 * 2^e, and each value is the integer
round(x / 2^e).  The forward uses gate and up as they came and returns what an
unsaved activation returns; the backward's gradients are those at the kept
values (error of a kept value: at most 2^e / 2, which is at most 1/127 of its
group's largest).  An infinity or NaN comes back from the copy as NaN.  gate
and up are not written and can be freed after the forward; gradients are new
tensors.

Arithmetic is fp32 with one rounding of each result.
"""
from __future__ import annotations

import torch

from forge_hip import _lib as L

ACTIVATIONS = {"silu": L.ACT_SILU, "gelu_tanh": L.ACT_GELU_TANH, "gelu_exact": L.ACT_GELU_ERF}
_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def _activation(name) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {name!r}")
    return ACTIVATIONS[name]


def _check_dtype(t: torch.Tensor) -> None:
    if t.dtype not in _DTYPES:
        raise TypeError(f"glu_act8 supports fp16, bf16, and fp32, got {t.dtype}")


def _check_pair(gate: torch.Tensor, up: torch.Tensor) -> None:
    if gate.dim() == 0 or gate.shape != up.shape:
        raise ValueError(f"gate and up must have the same shape, got {tuple(gate.shape)} and {tuple(up.shape)}")
    if gate.device != up.device:
        raise ValueError("gate and up must be on the same device")
    if gate.dtype != up.dtype:
        raise TypeError(f"gate and up must have the same dtype, got {gate.dtype} and {up.dtype}")
    _check_dtype(gate)
    L.require_gpu(gate)


def _rows(t: torch.Tensor):
    """(2-D view or copy of t with unit column stride, its row pitch)."""
    rows, cols = t.numel() // t.shape[-1] if t.shape[-1] else 0, t.shape[-1]
    if t.is_contiguous():
        return t, cols
    t = t.reshape(rows, cols)
    if cols > 1 and t.stride(1) != 1 or rows > 1 and t.stride(0) < cols:
        t = t.contiguous()
    return t, t.stride(0) if rows > 1 else cols


def _forward(gate, up, act, keep):
    cols = gate.shape[-1]
    rows = gate.numel() // cols if cols else 0
    gate, ld_gate = _rows(gate)
    up, ld_up = _rows(up)
    out = torch.empty((rows, cols), dtype=gate.dtype, device=gate.device)
    kept = torch.empty(L.forge_glu_act8_bytes(rows, cols), dtype=torch.uint8, device=gate.device) if keep else None
    if out.numel():
        with L.on_device(out):
            L.check(L.forge_glu_act8_fwd(L.dtype_code(out.dtype), act, gate.data_ptr(), ld_gate, up.data_ptr(), ld_up,
                                         out.data_ptr(), cols, L.ptr(kept), rows, cols, L.stream_of(out)),
                    "forge_glu_act8_fwd")
    return out, kept


def _backward(dout, kept, dtype, act, dgate, dup, ld_grad):
    """dgate, dup: [rows, cols] with rows ld_grad apart."""
    rows, cols = dgate.shape
    if dgate.numel() == 0:
        return
    dout, ld_dout = _rows(dout)
    with L.on_device(dout):
        L.check(L.forge_glu_act8_bwd(L.dtype_code(dtype), act, dout.data_ptr(), ld_dout, kept.data_ptr(),
                                     dgate.data_ptr(), dup.data_ptr(), ld_grad, rows, cols, L.stream_of(dout)),
                "forge_glu_act8_bwd")


class ForgeGLUAct8Function(torch.autograd.Function):
    """forward(ctx, gate, up, activation code); saves the 8-bit copy."""

    @staticmethod
    def forward(ctx, gate, up, act):
        out, kept = _forward(gate, up, act, keep=True)
        ctx.save_for_backward(kept)
        ctx.act = act
        return out.view(gate.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        (kept,) = ctx.saved_tensors
        cols = dout.shape[-1]
        rows = dout.numel() // cols if cols else 0
        dgate, dup = (torch.empty((rows, cols), dtype=dout.dtype, device=dout.device) for _ in range(2))
        _backward(dout, kept, dout.dtype, ctx.act, dgate, dup, cols)
        return dgate.view(dout.shape), dup.view(dout.shape), None


class ForgePackedGLUAct8Function(torch.autograd.Function):
    """forward(ctx, gate_up [..., 2 cols], activation code): gate and up side
    by side, and their gradients in one tensor."""

    @staticmethod
    def forward(ctx, gate_up, act):
        cols = gate_up.shape[-1] // 2
        out, kept = _forward(gate_up[..., :cols], gate_up[..., cols:], act, keep=True)
        ctx.save_for_backward(kept)
        ctx.act = act
        return out.view(*gate_up.shape[:-1], cols)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        (kept,) = ctx.saved_tensors
        cols = dout.shape[-1]
        rows = dout.numel() // cols if cols else 0
        grad = torch.empty((rows, 2 * cols), dtype=dout.dtype, device=dout.device)
        _backward(dout, kept, dout.dtype, ctx.act, grad[:, :cols], grad[:, cols:], 2 * cols)
        return grad.view(*dout.shape[:-1], 2 * cols), None


def glu_act8(gate: torch.Tensor, up: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """act(gate) * up for gate, up [..., cols] (fp16, bf16, fp32; any row
    pitch), activation "silu", "gelu_tanh" or "gelu_exact".  Where a gradient
    is wanted, gate and up are kept in 8 bits and not otherwise saved; without
    one nothing is kept."""
    act = _activation(activation)
    _check_pair(gate, up)
    if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad):
        return ForgeGLUAct8Function.apply(gate, up, act)
    L.refuse_tangents(gate, up)
    return _forward(gate, up, act, keep=False)[0].view(gate.shape)


def glu_act8_packed(gate_up: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """glu_act8 of the two halves of gate_up [..., 2 cols]."""
    act = _activation(activation)
    if gate_up.dim() == 0 or gate_up.shape[-1] % 2 != 0:
        raise ValueError(f"packed gate_up last dimension must be even, got shape {tuple(gate_up.shape)}")
    _check_dtype(gate_up)
    L.require_gpu(gate_up)
    if torch.is_grad_enabled() and gate_up.requires_grad:
        return ForgePackedGLUAct8Function.apply(gate_up, act)
    L.refuse_tangents(gate_up)
    cols = gate_up.shape[-1] // 2
    out, _ = _forward(gate_up[..., :cols], gate_up[..., cols:], act, keep=False)
    return out.view(*gate_up.shape[:-1], cols)


__all__ = ["ACTIVATIONS", "ForgeGLUAct8Function", "ForgePackedGLUAct8Function", "glu_act8", "glu_act8_packed"]
