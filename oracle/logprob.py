"""Token log-probabilities, preference loss and policy loss in float64 from
their formulas, with each loss's derivative by the log-probabilities."""
from __future__ import annotations

import torch

IGNORE = -100


def token_logps(logits, target, ignore=IGNORE, temperature=1.0):
    """log softmax(logits / temperature) at the targets, 0 where ignored."""
    z = logits.double() / temperature
    lp = z.log_softmax(-1).gather(-1, target.masked_fill(target == ignore, 0).unsqueeze(-1)).squeeze(-1)
    return torch.where(target == ignore, 0.0, lp)


def dlogits(logits, target, coef, ignore=IGNORE, temperature=1.0):
    """coef / temperature (onehot - softmax); zero rows where ignored."""
    p = (logits.double() / temperature).softmax(-1)
    hot = torch.zeros_like(p).scatter_(-1, target.masked_fill(target == ignore, 0).unsqueeze(-1), 1.0)
    c = torch.where(target == ignore, 0.0, coef.double() / temperature).unsqueeze(-1)
    return torch.where(c == 0, 0.0, c * (hot - p))


def preference(logps, kept, ref, beta, smoothing, kind, normalized, reduction):
    """logps, kept [2 P, S] -> (loss, sequences' log-probabilities, rewards,
    dloss/dlogps [2 P, S])."""
    n = kept.sum(-1).double().clamp(min=1) if normalized else torch.ones(len(logps), dtype=torch.float64)
    seq = torch.where(kept, logps, 0.0).sum(-1) / n
    over = seq - (0.0 if ref is None else ref.double())
    c, r = over.chunk(2)
    h = beta * (c - r)
    if kind == "sigmoid":
        log_s = torch.nn.functional.logsigmoid
        loss = -(1 - smoothing) * log_s(h) - smoothing * log_s(-h)
        d = beta * (-(1 - smoothing) * torch.sigmoid(-h) + smoothing * torch.sigmoid(h))
    elif kind == "hinge":
        loss, d = (1 - h).clamp(min=0), -beta * (h < 1).double()
    else:
        loss, d = (h / beta - 1 / (2 * beta)) ** 2, 2 * (h / beta - 1 / (2 * beta))
    if reduction == "mean":
        loss, d = loss.mean(), d / len(d)
    elif reduction == "sum":
        loss = loss.sum()
    coef = torch.where(kept, (torch.cat([d, -d]) / n).unsqueeze(-1), 0.0)
    return loss, seq, beta * over, coef


def policy(logps, kept, adv, old, ref, low, high, beta, reduction):
    """logps, kept, adv, old, ref [N, S] -> (loss, kl, dloss/dlogps)."""
    lp, adv = torch.where(kept, logps, 0.0), torch.where(kept, adv.double(), 0.0)
    ratio = torch.ones_like(lp) if old is None else torch.where(kept, lp - old.double(), 0.0).exp()
    free, held = ratio * adv, ratio.clamp(1 - low, 1 + high) * adv
    loss, d = -torch.minimum(free, held), torch.where(free <= held, -free, 0.0)
    kl = torch.zeros_like(lp)
    if ref is not None:
        f = torch.where(kept, ref.double() - lp, 0.0)
        kl = torch.expm1(f) - f
        loss, d = loss + beta * kl, d - beta * torch.expm1(f)
    tokens = kept.sum(-1).double()
    if reduction == "mean":
        w = torch.ones_like(lp) / tokens.sum().clamp(min=1)
    elif reduction == "sequence":
        w = torch.ones_like(lp) / tokens.clamp(min=1).unsqueeze(-1) / (tokens > 0).sum().clamp(min=1)
    else:
        w = torch.ones_like(lp)
    w = torch.where(kept, w, 0.0)
    return (loss * w).sum(), kl, d * w
