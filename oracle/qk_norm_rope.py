"""RMS norm of each head and RoPE, in float64 from the formulas, with the
closed-form gradients and, per element, the size of the terms that an fp32
evaluation adds up (what its rounding errors are relative to)."""
from __future__ import annotations

from typing import NamedTuple

import torch


class HeadResult(NamedTuple):
    out: torch.Tensor
    out_terms: torch.Tensor
    dx: torch.Tensor
    dx_terms: torch.Tensor
    dw: torch.Tensor
    dw_terms: torch.Tensor


def rotate(x, c, s):
    """Half-split rotation by angles whose cosines and sines are c, s [..., D/2]."""
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


def forward(x, w, c, s, eps, offset):
    """x [B, H, S, D] -> rope(rmsnorm(x) * (w + offset))."""
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return rotate(x * r * (w + offset), c, s)


def head_fwd_bwd(x, w, cos, sin, do, eps, offset) -> HeadResult:
    """All in float64: x, do [B, H, S, D]; w [D]; cos, sin [B or 1, S, D] rows
    of each token."""
    x, w, do, cos, sin = (t.double() for t in (x, w, do, cos, sin))
    half = x.shape[-1] // 2
    c, s = cos[..., :half].unsqueeze(1), sin[..., :half].unsqueeze(1)
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n, w1 = x * r, w + offset
    y = n * w1
    out_terms = rotate(y.abs(), c.abs(), -s.abs())
    out_terms = torch.cat([out_terms[..., :half], (y[..., half:] * c).abs() + (y[..., :half] * s).abs()], -1)
    dy = rotate(do, c, -s)
    lo, hi = do[..., :half].abs(), do[..., half:].abs()
    dy_terms = torch.cat([lo * c.abs() + hi * s.abs(), hi * c.abs() + lo * s.abs()], -1)
    g, g_terms = dy * w1, dy_terms * w1.abs()
    mean, mean_terms = (g * n).mean(-1, keepdim=True), (g_terms * n.abs()).mean(-1, keepdim=True)
    return HeadResult(rotate(y, c, s), out_terms, r * (g - n * mean), r * (g_terms + n.abs() * mean_terms),
                      (dy * n).sum((0, 1, 2)), (dy_terms * n.abs()).sum((0, 1, 2)))
