"""RMS norm with the residual's addition (csrc/add_rmsnorm.hip, add_rmsnorm_bwd.hip).

    h = x + residual                  (rounded to x's type: the residual stream)
    y = h rsqrt(mean h^2 + eps) (weight + offset)

One pass over x and the residual instead of two over x, the residual and h; y is
rounded once, after the weight.  `add_rmsnorm_int8` gives y in 8 bits with a scale for
each row, as int8_linear takes it: the integers round(127 t / max |t|) of t = h (weight +
offset), which do not depend on the norm, and the scale max |t| rstd / 127.
"""
from __future__ import annotations

from typing import Optional

import torch

from forge_hip import _lib as L
from kernels.int8.int8 import Int8Rows, _ld, _new_rows, _rows

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def _check(x, residual, weight, eps):
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    if weight.dim() != 1 or x.shape[-1] != weight.numel():
        raise ValueError(f"weight must be [{x.shape[-1]}], got {tuple(weight.shape)}")
    if x.dtype not in _DTYPES or weight.dtype not in _DTYPES:
        raise TypeError(f"x and weight must be fp16, bf16 or fp32, got {x.dtype} and {weight.dtype}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual {tuple(residual.shape)} does not match x {tuple(x.shape)}")
        if residual.dtype != x.dtype:
            raise TypeError(f"x and residual must have the same dtype, got {x.dtype} and {residual.dtype}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if weight.device != x.device or (residual is not None and residual.device != x.device):
        raise ValueError(f"every tensor must be on x's device {x.device}")
    L.require_gpu(x)


def _forward(x, residual, weight, eps, offset, want_rstd):
    x2 = _rows(x)
    rows, H = x2.shape
    r2 = None if residual is None else _rows(residual)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if want_rstd else None
    if x.numel():
        with L.on_device(x):
            L.check(L.forge_add_rmsnorm_fwd(L.dtype_code(x.dtype), L.dtype_code(weight.dtype), x2.data_ptr(), _ld(x2),
                                            L.ptr(r2), 0 if r2 is None else _ld(r2), weight.data_ptr(), L.ptr(h),
                                            y.data_ptr(), L.ptr(rstd), rows, H, eps, offset, L.stream_of(x)),
                    "forge_add_rmsnorm_fwd")
    return y, h, rstd


def _backward(dy, dh, h, weight, rstd, offset, need_dw):
    h2, dy2 = _rows(h), _rows(dy)
    dh2 = None if dh is None else _rows(dh)
    rows, H = h2.shape
    d = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    dw = torch.empty_like(weight) if need_dw else None
    if h.numel() == 0:
        return d, dw.zero_() if need_dw else None
    code = L.dtype_code(h.dtype)
    work = None
    if need_dw:
        work = torch.empty(L.forge_add_rmsnorm_bwd_workspace(code, rows, H), dtype=torch.uint8, device=h.device)
    with L.on_device(h):
        L.check(L.forge_add_rmsnorm_bwd(code, L.dtype_code(weight.dtype), dy2.data_ptr(), _ld(dy2), L.ptr(dh2),
                                        0 if dh2 is None else _ld(dh2), h2.data_ptr(), _ld(h2), weight.data_ptr(),
                                        rstd.data_ptr(), d.data_ptr(), L.ptr(dw), L.ptr(work), rows, H, offset,
                                        L.stream_of(h)),
                "forge_add_rmsnorm_bwd")
    return d, dw


class ForgeAddRMSNormFunction(torch.autograd.Function):
    """forward(ctx, x, residual, weight, eps, offset) -> (y, h), or y alone without a
    residual, on checked arguments; saves h (or x), the weight and rstd."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, offset):
        y, h, rstd = _forward(x, residual, weight, eps, offset, True)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.offset = offset
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        need_dw = ctx.needs_input_grad[2]
        if dy is None:  # only the residual stream goes on
            return dh, dh, torch.zeros_like(weight) if need_dw and dh is not None else None, None, None
        d, dw = _backward(dy, dh, h, weight, rstd, ctx.offset, need_dw)
        return d, d if ctx.needs_input_grad[1] else None, dw, None, None


def add_rmsnorm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                offset: float = 0.0):
    """(y, h): h = x + residual (x itself where residual is None), y its norm times weight +
    offset.  x and residual [..., H] of one type, the weight [H] of any (fp16, bf16, fp32).
    Gradients: x, residual (the same tensor), weight."""
    _check(x, residual, weight, eps)
    weight = weight.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        out = ForgeAddRMSNormFunction.apply(x, residual, weight, float(eps), float(offset))
        return (out, x) if residual is None else out
    L.refuse_tangents(*(t for t in (x, residual, weight) if t is not None))
    y, h, _ = _forward(x, residual, weight, float(eps), float(offset), False)
    return y, x if h is None else h


def add_rmsnorm_int8(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                     offset: float = 0.0):
    """(rows, h) as add_rmsnorm, y as Int8Rows.  For inference: raises where a gradient
    would be lost (a training step calls add_rmsnorm, and int8_linear rounds its y)."""
    _check(x, residual, weight, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        raise ValueError("add_rmsnorm_int8 has no gradient; call add_rmsnorm, and int8_linear on its result")
    L.refuse_tangents(*(t for t in (x, residual, weight) if t is not None))
    weight = weight.contiguous()
    x2 = _rows(x)
    r2 = None if residual is None else _rows(residual)
    rows, H = x2.shape
    h = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    q, scale = _new_rows(rows, H, x.device)
    if x.numel():
        with L.on_device(x):
            L.check(L.forge_add_rmsnorm_int8(L.dtype_code(x.dtype), L.dtype_code(weight.dtype), x2.data_ptr(), _ld(x2),
                                             L.ptr(r2), 0 if r2 is None else _ld(r2), weight.data_ptr(), L.ptr(h),
                                             q.data_ptr(), q.shape[1], scale.data_ptr(), rows, H, float(eps), float(offset),
                                             L.stream_of(x)),
                    "forge_add_rmsnorm_int8")
    else:
        scale.zero_()
    return Int8Rows._of(q, scale, x.shape, x.dtype), x if h is None else h


__all__ = ["ForgeAddRMSNormFunction", "add_rmsnorm", "add_rmsnorm_int8"]
