"""Clipped policy loss with a divergence term from the policy's logits
(csrc/logprob.hip), forward and backward."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch

from forge_hip import _lib as L
from . import _rows as R

_REDUCTIONS = {"mean": L.REDUCE_MEAN, "sum": L.REDUCE_SUM, "sequence": L.REDUCE_SEQUENCE}


@dataclass(frozen=True)
class PolicyLossOutput:
    """loss: fp32 scalar.  logps: the tokens' log-probabilities; kl: e^f - f -
    1 with f = ref_logps - logps (0 without ref_logps, infinite where f is);
    fp32 in the target's shape, 0 where it is ignored.  Only the loss carries a gradient."""

    loss: torch.Tensor
    logps: torch.Tensor
    kl: torch.Tensor


def _launch(x, target, adv, old, ref, clip_low, clip_high, kl_coef, temperature, reduction, ignore_index, dlogits,
            grad_scale=None):
    n, s, _ = x.shape
    f32 = {"dtype": torch.float32, "device": x.device}
    loss, logps, kl = torch.empty((), **f32), torch.empty((n, s), **f32), torch.empty((n, s), **f32)
    work = R.workspace(x)

    def strided(t):
        return (None, 0, 0) if t is None else (t.data_ptr(), *t.stride())

    with L.on_device(x):
        L.check(
            L.forge_policy_loss_scaled(*R.rows_args(x, target, ignore_index), temperature, *strided(adv), *strided(old),
                                       *strided(ref), clip_low, clip_high, kl_coef, reduction, L.ptr(grad_scale),
                                       loss.data_ptr(), logps.data_ptr(), kl.data_ptr(), L.ptr(dlogits),
                                       *((0, 0) if dlogits is None else dlogits.stride()[:2]), work.data_ptr(),
                                       L.stream_of(x)),
            "forge_policy_loss")
    return loss, logps, kl


class ForgePolicyLossFunction(torch.autograd.Function):
    """forward(ctx, logits [N, S, V], target [N, S], advantages, old_logps,
    ref_logps [N, S] or None, clip_low, clip_high, kl_coef, temperature,
    reduction, ignore_index, inplace, grad_scale) -> (loss, logps, kl).  The
    forward writes dloss/dlogits times grad_scale (one fp32 element, or None),
    over the logits with inplace; the backward hands that out, scaled by the
    incoming gradient / grad_scale where that is not 1."""

    @staticmethod
    def forward(ctx, x, target, adv, old, ref, clip_low, clip_high, kl_coef, temperature, reduction, ignore_index,
                inplace, grad_scale=None):
        ctx.dlogits = x.detach() if inplace else torch.empty(x.shape, dtype=x.dtype, device=x.device)
        loss, logps, kl = _launch(x, target, adv, old, ref, clip_low, clip_high, kl_coef, temperature, reduction,
                                  ignore_index, ctx.dlogits, grad_scale)
        ctx.grad_scale = grad_scale
        if inplace:
            torch.autograd.graph.increment_version(x)  # what else has saved the logits must not use them
        ctx.mark_non_differentiable(logps, kl)
        return loss, logps, kl

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _logps, _kl):
        d, ctx.dlogits = ctx.dlogits, None
        if d is None:
            raise RuntimeError("forge_policy_loss: the gradient has been handed out; the backward runs once")
        n, s, v = d.shape
        if d.numel():
            # scaled in place on the device where the scale is not 1: a 16-bit
            # gradient is rounded a second time then, as in forge_cross_entropy
            grad = grad.to(torch.float32).reshape(1)
            if ctx.grad_scale is not None:
                grad = grad / ctx.grad_scale
            sn, ss, _ = d.stride()
            if s == 1:
                parts = [(d, n, sn)]
            elif n == 1 or sn == s * ss:
                parts = [(d, n * s, ss)]
            else:
                parts = [(d[i], s, ss) for i in range(n)]
            with L.on_device(d):
                for part, rows, ld in parts:
                    L.check(
                        L.forge_ce_scale(L.dtype_code(d.dtype), part.data_ptr(), max(ld, v), rows, v, grad.data_ptr(),
                                         L.DTYPE_F32, L.stream_of(d)),
                        "forge_ce_scale")
        return (d,) + (None,) * 12


def _scale(grad_scale, logits) -> torch.Tensor:
    """One fp32 element of the call's own."""
    if not isinstance(grad_scale, torch.Tensor):
        if not 2.0 ** -126 <= grad_scale < 2.0 ** 127:
            raise ValueError(f"grad_scale must be positive and finite in fp32, got {grad_scale}")
        return torch.full((1,), float(grad_scale), dtype=torch.float32, device=logits.device)
    if grad_scale.numel() != 1:
        raise ValueError(f"grad_scale must have one element, got shape {tuple(grad_scale.shape)}")
    if not grad_scale.is_floating_point():
        raise TypeError(f"grad_scale must be floating point, got {grad_scale.dtype}")
    if grad_scale.device != logits.device:
        raise ValueError(f"grad_scale must be on the logits' device {logits.device}, got {grad_scale.device}")
    return grad_scale.detach().reshape(1).to(torch.float32, copy=True)


def forge_policy_loss(logits: torch.Tensor, target: torch.Tensor, advantages: torch.Tensor,
                      old_logps: Optional[torch.Tensor] = None, ref_logps: Optional[torch.Tensor] = None,
                      clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0,
                      reduction: str = "mean", ignore_index: int = -100, inplace: bool = False,
                      validate_targets: bool = False,
                      grad_scale: Union[None, float, torch.Tensor] = None) -> PolicyLossOutput:
    """Policy-gradient loss of sampled tokens.  logits [N, S, V] (fp16, bf16,
    fp32), target [N, S] with ignore_index on prompts and padding (their rows
    are not read, and get zero gradients; nothing else of them is read either).
    With logp the log-probability under softmax(logits / temperature), r =
    exp(logp - old_logps) (None: the policy itself, r = 1) and f = ref_logps -
    logp, a token's loss is
        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (e^f - f - 1).
    advantages: [N] (one of a sequence) or [N, S]; old_logps, ref_logps [N, S];
    kl_coef needs ref_logps, and ref_logps alone reports kl.
    reduction: "mean" over the kept tokens, "sequence" (the mean of each
    sequence's mean, over those that have tokens), or "sum"; 0 where nothing is
    kept.

    Where the logits want a gradient the forward computes it, over the logits'
    storage with inplace (forge_cross_entropy's contract) or into a new tensor,
    and the backward runs once.  That gradient is rounded to the logits' type
    before the incoming one is known: under loss scaling (fp16) pass the loss's
    scale as grad_scale (a number, or one element on the device), and what is
    rounded is the scaled gradient; the loss is returned unscaled, and a
    backward from scale * loss hands the gradient out as it is.  A target outside [0, V) makes the loss NaN;
    validate_targets=True raises IndexError instead (one host sync)."""
    R.check_logits(logits, target, temperature)
    if logits.dim() != 3:
        raise ValueError(f"logits must be [sequences, seq, vocab], got {tuple(logits.shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if not 0.0 <= clip_low <= 1.0 or not clip_high >= 0.0:
        raise ValueError(f"clip_low must be between 0 and 1 and clip_high not negative, got {clip_low} and {clip_high}")
    if kl_coef and ref_logps is None:
        raise ValueError("kl_coef needs ref_logps")
    if inplace:
        R.check_inplace(logits)
    shape = target.shape
    if advantages.dim() == 1:
        advantages = R.per_token(advantages, shape[:1], "advantages", logits).unsqueeze(1).expand(shape)
    else:
        advantages = R.per_token(advantages, shape, "advantages", logits)
    old = None if old_logps is None else R.per_token(old_logps, shape, "old_logps", logits)
    ref = None if ref_logps is None else R.per_token(ref_logps, shape, "ref_logps", logits)
    if grad_scale is not None:
        grad_scale = _scale(grad_scale, logits)
    L.require_gpu(logits)
    if validate_targets:
        R.check_targets(target, ignore_index, logits.shape[-1])
    x, t = R.three_d(logits), R.target_2d(target, 3)
    args = (advantages, old, ref, float(clip_low), float(clip_high), float(kl_coef), float(temperature),
            _REDUCTIONS[reduction], int(ignore_index))
    if torch.is_grad_enabled() and logits.requires_grad:
        return PolicyLossOutput(*ForgePolicyLossFunction.apply(x, t, *args, bool(inplace), grad_scale))
    L.refuse_tangents(logits)
    return PolicyLossOutput(*_launch(x, t, *args, None))


__all__ = ["ForgePolicyLossFunction", "PolicyLossOutput", "forge_policy_loss"]
