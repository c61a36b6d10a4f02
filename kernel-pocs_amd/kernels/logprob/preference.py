"""Preference loss over pairs of answers from the policy's logits
(csrc/logprob.hip), forward and backward."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from forge_hip import _lib as L
from . import _rows as R

_KINDS = {"sigmoid": L.PREF_SIGMOID, "hinge": L.PREF_HINGE, "ipo": L.PREF_IPO}
_REDUCTIONS = {"none": L.REDUCE_NONE, "mean": L.REDUCE_MEAN, "sum": L.REDUCE_SUM}


@dataclass(frozen=True)
class PreferenceLossOutput:
    """loss: fp32, a scalar, or [pairs] with reduction "none".  logps [2 pairs]:
    the answers' log-probabilities; rewards [2 pairs]: beta (logps -
    ref_logps).  Only the loss carries a gradient."""

    loss: torch.Tensor
    logps: torch.Tensor
    rewards: torch.Tensor


class ForgePreferenceLossFunction(torch.autograd.Function):
    """forward(ctx, logits [2 P, S, V], target [2 P, S], ref, beta, smoothing,
    kind, normalized, reduction, ignore_index, inplace) -> (loss, logps,
    rewards).  The forward reads the logits once; the backward reads them again
    and writes their gradient, over the logits themselves with inplace."""

    @staticmethod
    def forward(ctx, x, target, ref, beta, smoothing, kind, normalized, reduction, ignore_index, inplace):
        n, s, _ = x.shape
        f32 = {"dtype": torch.float32, "device": x.device}
        loss = torch.empty((n // 2,) if reduction == L.REDUCE_NONE else (), **f32)
        seq_logps, rewards = torch.empty(n, **f32), torch.empty(n, **f32)
        held, (state, logps, coef, work) = R.held(x)
        with L.on_device(x):
            L.check(
                L.forge_preference_fwd(*R.rows_args(x[: n // 2], target, ignore_index), L.ptr(ref), beta, smoothing, kind,
                                       int(normalized), reduction, loss.data_ptr(), seq_logps.data_ptr(),
                                       rewards.data_ptr(), coef, logps, state, work, L.stream_of(x)),
                "forge_preference_fwd")
        # with inplace the backward writes over the logits, so they are kept
        # outside autograd's version check, and checked here
        ctx.save_for_backward(target, held, *(() if inplace else (x,)))
        ctx.x, ctx.version = (x.detach(), x._version) if inplace else (None, 0)
        ctx.ignore_index, ctx.inplace = ignore_index, inplace
        ctx.mark_non_differentiable(seq_logps, rewards)
        return loss, seq_logps, rewards

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _logps, _rewards):
        target, held, *saved = ctx.saved_tensors
        x = ctx.x if ctx.inplace else saved[0]
        if x is None:
            raise RuntimeError("forge_preference_loss: the backward with inplace=True has written over the logits and "
                               "runs once")
        if ctx.inplace and x._version != ctx.version:
            raise RuntimeError("forge_preference_loss: the logits have been modified in place since the forward")
        grad = grad.to(torch.float32)
        out = R.gradient(x, target, ctx.ignore_index, 1.0, *R.held_addresses(held, *x.shape[:2]), (1, 0), grad,
                         grad.stride(0) if grad.dim() else 0, x.shape[0] // 2, out=x if ctx.inplace else None)
        if ctx.inplace:
            ctx.x = None
            torch.autograd.graph.increment_version(x)  # what else has saved the logits must not use them
        return (out,) + (None,) * 9


def forge_preference_loss(logits: torch.Tensor, target: torch.Tensor, ref_logps: Optional[torch.Tensor] = None,
                          beta: float = 0.1, label_smoothing: float = 0.0, loss_type: str = "sigmoid",
                          length_normalized: bool = False, reduction: str = "mean", ignore_index: int = -100,
                          inplace: bool = False, validate_targets: bool = False) -> PreferenceLossOutput:
    """Preference loss of P pairs.  logits [2 P, S, V] (fp16, bf16, fp32) and
    target [2 P, S]: the P chosen answers, then the P rejected ones in the same
    order; prompts and padding carry ignore_index (their rows are not read, and
    get zero gradients).  ref_logps [2 P]: the reference model's
    log-probabilities of the answers (sums, or means with length_normalized;
    None: no reference).  With pi the policy's, h = beta ((pi_c - ref_c) -
    (pi_r - ref_r)) and loss_type
        "sigmoid"  -(1 - e) log s(h) - e log s(-h), e = label_smoothing
        "hinge"    max(0, 1 - h)
        "ipo"      (h / beta - 1 / (2 beta))^2
    reduced over the pairs ("mean", "sum", "none").

    inplace: the backward writes dlogits over the logits' storage (as
    forge_cross_entropy does in its forward) and runs once.  A target outside
    [0, V) makes its pair's loss NaN; validate_targets=True raises IndexError
    instead (one host sync)."""
    R.check_logits(logits, target)
    if logits.dim() != 3 or logits.shape[0] < 2 or logits.shape[0] % 2:
        raise ValueError(f"logits must be [2 * pairs, seq, vocab], got {tuple(logits.shape)}")
    if loss_type not in _KINDS:
        raise ValueError(f"loss_type must be one of {sorted(_KINDS)}, got {loss_type!r}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if not beta > 0.0:
        raise ValueError(f"beta must be positive, got {beta}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must be between 0.0 and 1.0, got {label_smoothing}")
    if label_smoothing and loss_type != "sigmoid":
        raise ValueError("label_smoothing belongs to loss_type='sigmoid'")
    if inplace:
        R.check_inplace(logits)
    if ref_logps is not None:
        ref_logps = R.per_token(ref_logps, (logits.shape[0],), "ref_logps", logits).contiguous()
    L.require_gpu(logits)
    if validate_targets:
        R.check_targets(target, ignore_index, logits.shape[-1])
    return PreferenceLossOutput(*ForgePreferenceLossFunction.apply(
        R.three_d(logits), R.target_2d(target, 3), ref_logps, float(beta), float(label_smoothing), _KINDS[loss_type],
        bool(length_normalized), _REDUCTIONS[reduction], int(ignore_index), bool(inplace)))


__all__ = ["ForgePreferenceLossFunction", "PreferenceLossOutput", "forge_preference_loss"]
