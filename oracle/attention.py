"""Attention of one head of one sequence in float64, with its gradients, and the
sums of magnitudes from which tests derive their bounds.

    s = scale q k^T, p = softmax over the keys that a query sees, o = p v
    dv = p^T do, ds = p (do v^T - rowsum(do o)), dq = scale ds k, dk = scale ds^T q

Causal: query i sees key j where j <= i + len_k - len_q.  A query that sees no
key has o = 0, lse = -inf and no gradient."""
from __future__ import annotations

from types import SimpleNamespace

import torch

FLUSH = 2.0 ** -126  # v_exp_f32 returns 0 where the result is below it


def head_fwd_bwd(q, k, v, do, scale, causal, unit, tiny, tiny_bwd=None):
    """q, do [n, D]; k, v [m, D] (any floating type).  unit: the largest relative
    error of rounding to the kernels' operand type, tiny: its largest absolute one
    (half the spacing of its subnormals); tiny_bwd: that of the gradients' p and ds,
    where they are held as multiples.

    Returns o, lse, dq, dk, dv and for each x an x_err: how far a computation may be
    that keeps s, sums and statistics in fp32, and rounds p, ds and o to that type."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    n, m = q.shape[0], k.shape[0]
    u32 = 2.0 ** -24
    tiny_bwd = tiny if tiny_bwd is None else tiny_bwd
    sees = torch.ones(n, m, dtype=torch.bool)
    if causal:
        sees = sees.tril(m - n)
    s = (scale * q @ k.T).masked_fill(~sees, float("-inf"))
    lse = torch.logsumexp(s, -1) if m else torch.full((n,), float("-inf"), dtype=torch.float64)
    p = torch.where(sees, torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse).unsqueeze(1)), 0.0)
    o = p @ v
    # relative error of a probability: its exponent in fp32 (D products, the statistics, log2(e)) and exp
    depth = q.shape[1] + 8
    mag = scale * q.abs() @ k.abs().T
    rel = torch.where(sees, (mag + mag.amax(-1, keepdim=True) if m else mag) * depth * u32 + (m + 16) * u32, 0.0)
    p_err = p * (unit + rel) + (tiny + FLUSH) * sees
    sum_err = p_err @ v.abs() + (rel * p).sum(-1, keepdim=True) * (p @ v.abs())
    o_err = sum_err + o.abs() * unit + tiny
    lse_err = (rel * p).sum(-1) + (lse.abs().nan_to_num(0.0, 0.0, 0.0) + 1) * 8 * u32
    dp = do @ v.T
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dp_mag = do.abs() @ v.abs().T
    # delta is formed of o before its rounding, but for half a 254th of a step (a step: twice the largest
    # rounding, unit |o| at least, or tiny)
    half_part = (o.abs() * unit + tiny) / 254
    delta_err = (do.abs() * (sum_err + half_part + depth * u32 * o.abs())).sum(-1, keepdim=True)
    # (a probability below the smallest normal of fp32 is 0: off by FLUSH, and ds by that times its other factor)
    ds_err = p * (delta_err + dp_mag * depth * u32) + ds.abs() * (unit + 3 * rel) + (tiny_bwd + FLUSH * (dp - delta).abs()) * sees
    pv_err = p * (unit + 3 * rel) + (tiny_bwd + FLUSH) * sees
    # fp32 sums over up to n or m terms
    acc_n, acc_m = (n + 16) * u32, (m + 16) * u32
    dq, dk, dv = scale * ds @ k, scale * ds.T @ q, p.T @ do
    dq_err = scale * (ds_err + ds.abs() * acc_m) @ k.abs() + dq.abs() * unit + tiny
    dk_err = scale * (ds_err + ds.abs() * acc_n).T @ q.abs()  # (summed over heads before it is rounded)
    dv_err = (pv_err + p * acc_n).T @ do.abs()
    return SimpleNamespace(o=o, lse=lse, dq=dq, dk=dk, dv=dv, o_err=o_err, lse_err=lse_err, dq_err=dq_err,
                           dk_err=dk_err, dv_err=dv_err)


def packed_fwd_bwd(q, k, v, do, cu_q, cu_k, scale, causal, unit, tiny, tiny_bwd=None):
    """The same of packed sequences: q, do [T, H, D], k, v [T_k, Hkv, D] on the CPU, offsets as
    lists; rows outside the sequences are zeros (lse -inf)."""
    T, H, D = q.shape
    kv = k.shape[1]
    r = SimpleNamespace(o=torch.zeros(T, H, D).double(), lse=torch.full((T, H), float("-inf")).double(),
                        dq=torch.zeros(T, H, D).double(), dk=torch.zeros(k.shape).double(),
                        dv=torch.zeros(k.shape).double())
    err = {n + "_err": torch.zeros_like(getattr(r, n)) for n in ("o", "lse", "dq", "dk", "dv")}
    for i in range(len(cu_q) - 1):
        a, b = slice(cu_q[i], cu_q[i + 1]), slice(cu_k[i], cu_k[i + 1])
        for h in range(H):
            g = h * kv // H
            x = head_fwd_bwd(q[a, h], k[b, g], v[b, g], do[a, h], scale, causal, unit, tiny, tiny_bwd)
            for n in ("o", "lse", "dq"):
                getattr(r, n)[a, h] = getattr(x, n)
                err[n + "_err"][a, h] = getattr(x, n + "_err")
            for n in ("dk", "dv"):
                getattr(r, n)[b, g] += getattr(x, n)
                err[n + "_err"][b, g] += getattr(x, n + "_err")
    for n in ("dk", "dv"):
        err[n + "_err"] += getattr(r, n).abs() * unit + tiny
    r.__dict__.update(err)
    return r
