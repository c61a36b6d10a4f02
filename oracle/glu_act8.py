"""Gated activation with gate and up kept in 8 bits for the backward pass, in
float64 from the definition."""
from __future__ import annotations

import math

import torch

GROUP = 32


def kept(x: torch.Tensor) -> torch.Tensor:
    """The values that the 8-bit copy of x [rows, cols] stands for (float64):
    groups of 32 along a row, the least power of two 2^e (e >= -126) with
    |x| <= 127 * 2^e among the finite ones, round(x / 2^e) * 2^e; NaN where x
    is not finite."""
    x = x.double()
    rows, cols = x.shape
    g = torch.nn.functional.pad(x, (0, -cols % GROUP)).reshape(rows, -1, GROUP)
    finite = g.isfinite()
    m = torch.where(finite, g.abs(), 0.0).amax(-1, keepdim=True)
    e = torch.full(m.shape, -126, dtype=torch.int32)
    for _ in range(260):  # the definition, one exponent at a time
        e = e + (m > 127.0 * torch.ldexp(torch.ones_like(m), e)).to(torch.int32)
    q = torch.where(finite, torch.ldexp(torch.round(torch.ldexp(g, -e)), e), float("nan"))
    return q.reshape(rows, -1)[:, :cols]


def act_and_slope(x: torch.Tensor, activation: str):
    x = x.double()
    if activation == "silu":
        s = torch.sigmoid(x)
        return x * s, s * (1 + x * (1 - s))
    if activation == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        u = a * (x + 0.044715 * x ** 3)
        # (1 + tanh u) / 2 and (1 - tanh u) / 2, which cancel in float64 too where tanh u nears -1 or 1
        up, down = torch.sigmoid(2 * u), torch.sigmoid(-2 * u)
        return x * up, up + 2 * x * up * down * a * (1 + 3 * 0.044715 * x * x)
    cdf = 0.5 * torch.special.erfc(-x / math.sqrt(2))
    return x * cdf, cdf + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def fwd_bwd(gate, up, dout, activation):
    """(out, dgate, dup) in float64 for [rows, cols] inputs."""
    out = act_and_slope(gate, activation)[0] * up.double()
    g, u, d = kept(gate), kept(up), dout.double()
    act, slope = act_and_slope(g, activation)
    return out, d * u * slope, d * act
