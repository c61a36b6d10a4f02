"""What the log-probability entry points share: checks and layouts of logits
[..., V] with one target a row, and the launches of csrc/logprob.hip."""
from __future__ import annotations

import torch

from forge_hip import _lib as L

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def check_logits(logits: torch.Tensor, target: torch.Tensor, temperature: float = 1.0) -> None:
    if logits.dim() < 1 or logits.shape[:-1] != target.shape:
        raise ValueError(f"logits [..., V] need one target a row, got {tuple(logits.shape)} and {tuple(target.shape)}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be fp16, bf16 or fp32, got {logits.dtype}")
    if target.dtype.is_floating_point or target.dtype.is_complex or target.dtype == torch.bool:
        raise TypeError(f"target must be an integer tensor, got {target.dtype}")
    if logits.shape[-1] == 0 and target.numel():
        raise ValueError("logits have no columns")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must be between 1e-6 and 1e6, got {temperature}")
    if target.device != logits.device:
        raise ValueError(f"target must be on the logits' device {logits.device}, got {target.device}")


def check_targets(target: torch.Tensor, ignore_index: int, vocab: int) -> None:
    """IndexError unless every target is ignore_index or in [0, vocab) (one
    host sync)."""
    if target.numel() == 0:
        return
    lo, hi = (int(v) for v in torch.aminmax(torch.where(target == ignore_index, 0, target)))
    if lo < 0 or hi >= vocab:
        raise IndexError(f"targets must be {ignore_index} or lie in [0, {vocab}); got min {lo}, max {hi}")


def per_token(t: torch.Tensor, shape, name: str, logits: torch.Tensor) -> torch.Tensor:
    """An fp32 per-token input of the given leading shape (a view where it can
    be one: expanded tensors stay expanded)."""
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_floating_point():
        raise TypeError(f"{name} must be floating point, got {t.dtype}")
    if t.device != logits.device:
        raise ValueError(f"{name} must be on the logits' device {logits.device}, got {t.device}")
    return t.detach().to(torch.float32)


def three_d(logits: torch.Tensor) -> torch.Tensor:
    """logits as [N, S, V] with a unit column stride; a view unless the leading
    dimensions cannot be two strides or columns are not adjacent."""
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    if logits.dim() == 1:
        return logits.view(1, 1, -1)
    if logits.dim() == 2:
        return logits.unsqueeze(0)
    if logits.dim() == 3:
        return logits
    return logits.flatten(0, -3)


def two_d(t: torch.Tensor, dim: int) -> torch.Tensor:
    """A per-token tensor of logits with `dim` dimensions as [N, S]."""
    if dim == 1:
        return t.reshape(1, 1)
    if dim == 2:
        return t.unsqueeze(0)
    if dim == 3:
        return t
    return t.flatten(0, -2)


def target_2d(target: torch.Tensor, dim: int) -> torch.Tensor:
    return two_d(target.to(torch.int64), dim)


def check_inplace(logits: torch.Tensor) -> None:
    """The gradient can be written over [N, S, V] logits only where they are an
    operation's result, columns are adjacent and no two elements share memory."""
    base = logits._base
    if logits.requires_grad and (logits.is_leaf or base is not None and base.is_leaf and base.requires_grad):
        raise ValueError("inplace needs logits that are not a leaf, nor a view of one: their gradient would be themselves")
    (n, s, v), (sn, ss, sv) = logits.shape, logits.stride()
    inner, outer = ((s, ss), (n, sn)) if ss <= sn else ((n, sn), (s, ss))
    ok = v <= 1 or sv == 1
    reach = v
    for size, stride in (inner, outer):
        if size > 1:
            ok = ok and stride >= reach
            reach = stride * size
    if not ok or (v == 1 and sv != 1):
        raise ValueError(f"inplace needs logits with adjacent columns and rows of their own, got strides {(sn, ss, sv)}")


def rows_args(x: torch.Tensor, target: torch.Tensor, ignore_index: int):
    """The leading arguments of every entry point (x [N, S, V], target [N, S])."""
    n, s, v = x.shape
    return (L.dtype_code(x.dtype), x.data_ptr(), x.stride(0), x.stride(1), n, s, v, target.data_ptr(),
            target.stride(0), target.stride(1), int(ignore_index))


def workspace(x: torch.Tensor) -> torch.Tensor:
    return torch.empty(L.forge_logp_workspace(L.dtype_code(x.dtype), *x.shape), dtype=torch.uint8, device=x.device)


def held(x: torch.Tensor):
    """One buffer of a forward whose backward reads the logits again: each
    row's state (2 floats) and log-probability, each sequence's coefficient,
    and the forward's workspace behind them -> (buffer, the four addresses)."""
    n, s, _ = x.shape
    rows = -(-n * s // 4) * 4
    logps = 8 * rows
    coef = logps + 4 * rows
    work = coef + -(-n // 4) * 16
    buf = torch.empty(work + L.forge_logp_workspace(L.dtype_code(x.dtype), *x.shape), dtype=torch.uint8, device=x.device)
    at = buf.data_ptr()
    return buf, (at, at + logps, at + coef, at + work)


def gradient(x, target, ignore_index, temperature, state, logps, coef, coef_strides, up, up_stride, up_count, out=None):
    """dlogits of coef (times up) times each row's log-probability, dense
    unless `out` (the logits themselves) takes it.  state, logps and coef are
    addresses."""
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel():
        with L.on_device(x):
            L.check(
                L.forge_token_logps_bwd(*rows_args(x, target, ignore_index), temperature, logps, state, coef,
                                        *coef_strides, L.ptr(up), up_stride, up_count, out.data_ptr(), out.stride(0),
                                        out.stride(1), L.stream_of(x)),
                "forge_token_logps_bwd")
    return out


def held_addresses(buf: torch.Tensor, n: int, s: int):
    """(state, log-probabilities, coefficients) of a buffer of `held`."""
    rows, at = -(-n * s // 4) * 4, buf.data_ptr()
    return at, at + 8 * rows, at + 12 * rows
