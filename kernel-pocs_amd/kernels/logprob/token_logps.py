"""Log-probabilities of target tokens (csrc/logprob.hip): what a reference or
sampling policy's pass returns for the preference and policy losses, and a
differentiable building block for losses of one's own."""
from __future__ import annotations

import torch

from forge_hip import _lib as L
from . import _rows as R


def _forward(x, target, ignore_index, temperature, keep):
    n, s, _ = x.shape
    logps = torch.empty((n, s), dtype=torch.float32, device=x.device)
    state = torch.empty((n, s, 2), dtype=torch.float32, device=x.device) if keep else None
    if logps.numel():
        work = R.workspace(x)
        with L.on_device(x):
            L.check(
                L.forge_token_logps_fwd(*R.rows_args(x, target, ignore_index), temperature, logps.data_ptr(),
                                        L.ptr(state), work.data_ptr(), L.stream_of(x)),
                "forge_token_logps_fwd")
    return logps, state


class ForgeTokenLogpsFunction(torch.autograd.Function):
    """forward(ctx, logits [N, S, V], target [N, S], ignore_index,
    temperature); saves the logits and two fp32 values a row, and the backward
    reads the logits again."""

    @staticmethod
    def forward(ctx, x, target, ignore_index, temperature):
        logps, state = _forward(x, target, ignore_index, temperature, keep=True)
        ctx.save_for_backward(x, target, logps, state)
        ctx.ignore_index, ctx.temperature = ignore_index, temperature
        return logps

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, target, logps, state = ctx.saved_tensors
        grad = grad.to(torch.float32)
        return (R.gradient(x, target, ctx.ignore_index, ctx.temperature, state.data_ptr(), logps.data_ptr(),
                           grad.data_ptr(), grad.stride(), None, 0, 1), None, None, None)


def forge_token_logps(logits: torch.Tensor, target: torch.Tensor, ignore_index: int = -100, temperature: float = 1.0,
                      validate_targets: bool = False) -> torch.Tensor:
    """log softmax(logits / temperature) at each target, fp32 in the target's
    shape; 0 where the target is ignore_index (those rows are not read).

    logits [..., V] (fp16, bf16, fp32) in any row strides, target [...]
    integers.  To score the next token, shift the targets and leave the logits
    whole: a slice logits[:, :-1] makes autograd pad its gradient again.
    A target outside [0, V) gives NaN for its row; validate_targets=True raises
    IndexError instead (one host sync).  Differentiable in the logits; a row
    whose incoming gradient is 0 gets zeros."""
    R.check_logits(logits, target, temperature)
    L.require_gpu(logits)
    if validate_targets:
        R.check_targets(target, ignore_index, logits.shape[-1])
    x, t = R.three_d(logits), R.target_2d(target, logits.dim())
    if torch.is_grad_enabled() and logits.requires_grad:
        logps = ForgeTokenLogpsFunction.apply(x, t, int(ignore_index), float(temperature))
    else:
        L.refuse_tangents(logits)
        logps, _ = _forward(x, t, int(ignore_index), float(temperature), keep=False)
    return logps.reshape(target.shape)


__all__ = ["ForgeTokenLogpsFunction", "forge_token_logps"]
