"""Rows in 8 bits and products of them, in exact arithmetic (64 bits)."""
from __future__ import annotations

import torch


def quantize(t):
    """(integers, a / 127) of the rows of t: round(127 t / a), half to even, a = max |t|."""
    t = t.double()
    a = t.abs().amax(-1, keepdim=True) if t.shape[-1] else t.new_zeros(*t.shape[:-1], 1)
    q = torch.where(a > 0, torch.round(127 * t / torch.where(a > 0, a, 1.0)), 0.0)
    return q.to(torch.int64), (a / 127).squeeze(-1)


def linear(q, scale, w, w_scale, bias=None):
    """((sum_k q w) scale w_scale + bias, the magnitudes of both terms)."""
    y = (q.double() @ w.double().T) * scale.double().unsqueeze(1) * w_scale.double()
    b = 0.0 if bias is None else bias.double()
    return y + b, y.abs() + abs(b)
