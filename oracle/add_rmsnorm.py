"""RMS norm with the residual's addition in float64, its gradients, and the sums of
magnitudes that bound a computation in fp32."""
from __future__ import annotations

from types import SimpleNamespace

import torch


def fwd_bwd(x, residual, weight, dy, dh, eps, offset):
    """x, residual (or None), dy, dh (or None): [rows, H]; y and d unrounded, h rounded to x's
    type (the stream is stored in it, and normed as stored)."""
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    f, w = h.double(), weight.double() + offset
    rstd = 1.0 / torch.sqrt(f.square().mean(-1, keepdim=True) + eps)
    n = f * rstd
    r = SimpleNamespace(h=h, y=n * w, rstd=rstd.squeeze(-1))
    if dy is None:
        return r
    dy = dy.double()
    g = dy * w
    s = 0.0 if dh is None else dh.double()
    r.d = s + rstd * (g - n * (g * n).mean(-1, keepdim=True))
    r.d_terms = abs(s) + rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    r.dw = (dy * n).sum(0)
    r.dw_terms = (dy * n).abs().sum(0)
    return r
