"""The operators of a preference or policy fine-tuning step whose speed is measured.

Beside the LoRA layers and the cross-entropy of perf/cases.py such a step runs the norm and rotation
of queries and keys, a gated activation that keeps its inputs in 8 bits for the backward pass, the
log-probabilities of the tokens (a reference model's, or those of sampled tokens), and the loss: a
preference loss over pairs of answers, or a clipped policy loss with a KL term.

Where `own` is false the operators run in their plain form, elementary operations in 32 bits (sums
over a sequence and over a vocabulary in 64); where it is true they run through the framework.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORE = -100
EPS = 1e-6
GROUP = 32  # values that share one scale in an activation kept in 8 bits


def _own():
    """The framework's entry points."""
    root = str(Path.cwd() / "kernel-pocs_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from forge.kernels.glu_act8 import glu_act8, glu_act8_packed
    from forge.kernels.logprob import forge_policy_loss, forge_preference_loss, forge_token_logps
    from forge.kernels.rope import apply_qk_norm_rope

    return {"qk": apply_qk_norm_rope, "logps": forge_token_logps, "preference": forge_preference_loss,
            "policy": forge_policy_loss, "glu": glu_act8, "glu_packed": glu_act8_packed}


_calls = {}


def _call(name):
    if not _calls:
        _calls.update(_own())
    return _calls[name]


def listed():
    return [
        # one step of serving: 16 sequences at far positions, one token each
        {"name": "qk_decode", "op": "qk", "batch": 16, "seq": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "positions": True, "offset": 0.0, "packed": True, "train": False, "dtype": "bf16"},
        # a training batch whose q and k are columns of one projection's output
        {"name": "qk_train", "op": "qk", "batch": 4, "seq": 4096, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "positions": False, "offset": 0.0, "packed": True, "train": True, "dtype": "bf16"},
        # packed sequences of an odd length in fp32, weights stored as their difference from one
        {"name": "qk_odd_fp32", "op": "qk", "batch": 3, "seq": 1003, "heads": 32, "kv_heads": 8, "head_dim": 64,
         "positions": True, "offset": 1.0, "packed": False, "train": True, "dtype": "fp32"},
        # log-probabilities of the tokens that one serving step has sampled
        {"name": "logps_step", "op": "logps", "seqs": 16, "seq": 1, "vocab": 128256, "temperature": 0.7,
         "train": False, "dtype": "bf16"},
        # a reference model's log-probabilities of a batch of answers
        {"name": "logps_batch", "op": "logps", "seqs": 4, "seq": 2048, "vocab": 128256, "temperature": 1.0,
         "train": False, "dtype": "bf16"},
        # two pairs of short answers over a 32k vocabulary
        {"name": "preference_short", "op": "preference", "seqs": 4, "seq": 128, "vocab": 32000, "kind": "sigmoid",
         "smoothing": 0.0, "normalized": False, "dtype": "bf16"},
        # two pairs of long answers over a 128k vocabulary
        {"name": "preference", "op": "preference", "seqs": 4, "seq": 2048, "vocab": 128256, "kind": "sigmoid",
         "smoothing": 0.1, "normalized": False, "dtype": "bf16"},
        # a small group of short answers
        {"name": "policy_short", "op": "policy", "seqs": 8, "seq": 64, "vocab": 32000, "temperature": 1.0,
         "kl": 0.04, "old": True, "reduction": "mean", "dtype": "bf16"},
        # a full batch of policy training
        {"name": "policy", "op": "policy", "seqs": 8, "seq": 1024, "vocab": 128256, "temperature": 1.0,
         "kl": 0.04, "old": True, "reduction": "mean", "dtype": "bf16"},
        # fp32 logits of an odd vocabulary, means taken over each sequence
        {"name": "policy_odd_fp32", "op": "policy", "seqs": 3, "seq": 211, "vocab": 50257, "temperature": 0.9,
         "kl": 0.0, "old": True, "reduction": "sequence", "dtype": "fp32"},
        # the gated activation of a full training batch
        {"name": "glu", "op": "glu", "act": "silu", "rows": 8192, "cols": 14336, "packed": False, "dtype": "bf16"},
        # a short batch of an odd width, gate and up side by side in one buffer
        {"name": "glu_odd", "op": "glu", "act": "gelu_tanh", "rows": 333, "cols": 4097, "packed": True, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm: as often odd as it comes."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


VOCABS = [32000, 50257, 128256, 151936, 256000]
MOST_LOGITS = 8192 * 128256 * 2  # bytes of the largest listed logits


def draw(rng):
    op = rng.choice(["qk", "qk", "logps", "preference", "preference", "policy", "policy", "glu", "glu"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "qk":
        heads, kv, dim = rng.choice([(32, 8, 128), (16, 8, 128), (32, 32, 128), (32, 8, 64), (8, 4, 256), (14, 2, 96)])
        train = rng.random() < 0.7
        batch = rng.choice([1, 2, 3, 4])
        most = 4 * 4096 * 40 * 128 * 2 // (batch * (heads + kv) * dim * BYTES[dtype])
        return {"op": op, "batch": batch, "seq": _log(rng, 16 if train else 1, min(8192, most)), "heads": heads,
                "kv_heads": kv, "head_dim": dim, "positions": rng.random() < 0.5, "offset": rng.choice([0.0, 1.0]),
                "packed": rng.random() < 0.5, "train": train, "dtype": dtype}
    if op == "glu":
        cols = rng.choice([5632, 9216, 11008, 14336, _log(rng, 500, 16000)])
        most = 8192 * 14336 * 2 // (cols * BYTES[dtype])
        return {"op": op, "act": rng.choice(["silu", "silu", "gelu_tanh", "gelu_exact"]),
                "rows": _log(rng, 16, min(8192, most)), "cols": cols, "packed": rng.random() < 0.5, "dtype": dtype}
    vocab = rng.choice(VOCABS + [_log(rng, 1000, 256000)])
    tokens = MOST_LOGITS // (vocab * BYTES[dtype])
    seqs = rng.choice([2, 4, 6]) if op == "preference" else rng.choice([1, 3, 4, 8])
    # a scoring call goes down to one token, a training batch has some
    case = {"op": op, "seqs": seqs, "seq": _log(rng, 1 if op == "logps" else 24, min(4096, tokens // seqs)),
            "vocab": vocab, "dtype": dtype}
    if op == "preference":
        return {**case, "kind": rng.choice(["sigmoid", "sigmoid", "ipo"]), "smoothing": rng.choice([0.0, 0.1]),
                "normalized": rng.random() < 0.3}
    case["temperature"] = rng.choice([1.0, 1.0, 0.7])
    if op == "logps":
        return {**case, "train": rng.random() < 0.3}
    return {**case, "kl": rng.choice([0.0, 0.04]), "old": rng.random() < 0.8,
            "reduction": rng.choice(["mean", "sequence", "sum"])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _answers(case):
    """Where each sequence's answer begins (after its prompt) and ends (before its padding)."""
    n, s = case["seqs"], case["seq"]
    if s < 8:
        return [(0, s)] * n
    return [(int(s * (0.1 + 0.25 * (0.5 + 0.5 * math.sin(3.0 * i)))), s - int(s * 0.2 * (0.5 + 0.5 * math.cos(2.0 * i))))
            for i in range(n)]


class _Draws:
    """Seeded tensors on the GPU."""

    def __init__(self, case, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = DTYPES[case["dtype"]]

    def normal(self, *shape, std=1.0, dtype=None):
        t = torch.empty(shape, dtype=dtype or self.dtype, device="cuda")
        return t.normal_(0.0, std, generator=self.g)


def _qk_inputs(case, seed):
    d = _Draws(case, seed)
    b, s, h, kv, dim = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "head_dim"))
    if case["packed"]:  # columns of one [B, S, (heads + 2 kv_heads) * head_dim] projection
        qkv = d.normal(b, s, h + 2 * kv, dim)
        q, k = qkv[:, :, :h].transpose(1, 2), qkv[:, :, h:h + kv].transpose(1, 2)
    else:
        q, k = d.normal(b, s, h, dim).transpose(1, 2), d.normal(b, s, kv, dim).transpose(1, 2)
    t = {"q": q, "k": k, "q_weight": d.normal(dim, std=0.1).add_(1.0 - case["offset"]),
         "k_weight": d.normal(dim, std=0.1).add_(1.0 - case["offset"])}
    rows = s
    if case["positions"]:  # packed sequences that begin again, or a serving step's far positions
        rows = max(s, 4096)
        if s == 1:
            t["positions"] = torch.randint(0, rows, (b, 1), device="cuda", generator=d.g)
        else:
            cut = s // 3 + 1
            t["positions"] = (torch.arange(s, device="cuda") % cut).expand(b, s).contiguous()
    inv = 1.0 / 500000.0 ** (torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    ang = torch.arange(rows, device="cuda", dtype=torch.float64).unsqueeze(1) * inv
    ang = torch.cat([ang, ang], 1)
    t["cos"], t["sin"] = ang.cos().to(d.dtype).unsqueeze(0), ang.sin().to(d.dtype).unsqueeze(0)
    if case["train"]:  # gradients come back from attention as dense [B, heads, S, head_dim]
        t["dq"], t["dk"] = d.normal(b, h, s, dim), d.normal(b, kv, s, dim)
    return t


def _token_logps(logits, target, temperature):
    """Log-probabilities of the targets, a sequence at a time, to place a sampler's and a reference model's near them."""
    rows = [(x.float() / temperature).log_softmax(-1).gather(-1, y.clamp(min=0).unsqueeze(-1)).squeeze(-1)
            for x, y in zip(logits, target)]
    return torch.stack(rows).masked_fill_(target == IGNORE, 0.0)


def _logits_inputs(case, seed):
    d = _Draws(case, seed)
    n, s, v = case["seqs"], case["seq"], case["vocab"]
    logits = d.normal(n, s, v, std=2.0)
    target = torch.randint(0, v, (n, s), device="cuda", generator=d.g)
    # a trained model gives most of its tokens a fair share
    logits.scatter_add_(-1, target.unsqueeze(-1), d.normal(n, s, 1, std=2.0).add_(8.0))
    at, (begin, end) = torch.arange(s, device="cuda"), torch.tensor(_answers(case), device="cuda").T.unsqueeze(-1)
    target.masked_fill_((at < begin) | (at >= end), IGNORE)
    t = {"logits": logits, "target": target}
    if case["op"] == "logps":
        if case["train"]:
            t["dlogps"] = d.normal(n, s, dtype=torch.float32)
        return t
    logps = _token_logps(logits, target, case.get("temperature", 1.0))
    if case["op"] == "preference":  # the reference model's log-probabilities of whole answers, from its own pass
        whole = logps.double().sum(-1)
        whole = whole + d.normal(n, std=3.0, dtype=torch.float32)
        if case["normalized"]:
            whole = whole / (target != IGNORE).sum(-1)
        t["ref_logps"] = whole.float()
        return t
    if case["old"]:
        t["old_logps"] = logps + d.normal(n, s, std=0.15, dtype=torch.float32)
    if case["kl"]:
        t["ref_logps"] = logps + d.normal(n, s, std=0.3, dtype=torch.float32)
    # right or wrong answers against a running baseline
    right = torch.rand(n, device="cuda", generator=d.g) < 0.6
    t["advantages"] = right.float() - 0.137
    return t


def _glu_inputs(case, seed):
    d = _Draws(case, seed)
    rows, cols = case["rows"], case["cols"]
    if case["packed"]:
        t = {"gate_up": d.normal(rows, 2 * cols)}
    else:
        t = {"gate": d.normal(rows, cols), "up": d.normal(rows, cols)}
    t["dout"] = d.normal(rows, cols)
    return t


def _inputs(case, seed):
    return {"qk": _qk_inputs, "glu": _glu_inputs}.get(case["op"], _logits_inputs)(case, seed)


def _trained(case):
    """The names of the inputs whose gradients the pass returns."""
    if case["op"] == "qk":
        return ["q", "k", "q_weight", "k_weight"] if case["train"] else []
    if case["op"] == "glu":
        return ["gate_up"] if case["packed"] else ["gate", "up"]
    return ["logits"] if case.get("train", True) else []


def prepare(case, seed):
    t = _inputs(case, seed)
    for n in _trained(case):
        t[n].requires_grad_(True)
    return case, t


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case, t = state
    return (_run_own if own else _run_plain)(case, t)


def _run_own(case, t):
    op = case["op"]
    leaves = [t[n] for n in _trained(case)]
    if op == "qk":
        out = _call("qk")(t["q"], t["k"], t["q_weight"], t["k_weight"], t["cos"], t["sin"],
                          positions=t.get("positions"), eps=EPS, offset=case["offset"])
        if not case["train"]:
            return out
        return (*out, *torch.autograd.grad(out, leaves, (t["dq"], t["dk"])))
    if op == "logps":
        out = _call("logps")(t["logits"], t["target"], temperature=case["temperature"])
        return (out, *torch.autograd.grad(out, leaves, t["dlogps"])) if case["train"] else (out,)
    if op == "preference":
        smoothing = case["smoothing"] if case["kind"] == "sigmoid" else 0.0  # the other losses have none
        o = _call("preference")(t["logits"], t["target"], t["ref_logps"], beta=0.1, label_smoothing=smoothing,
                                loss_type=case["kind"], length_normalized=case["normalized"])
        return (o.loss, o.logps, o.rewards, *torch.autograd.grad(o.loss, leaves))
    if op == "policy":
        o = _call("policy")(t["logits"], t["target"], t["advantages"], old_logps=t.get("old_logps"),
                            ref_logps=t.get("ref_logps"), clip_low=0.2, clip_high=0.28, kl_coef=case["kl"],
                            temperature=case["temperature"], reduction=case["reduction"])
        return (o.loss, o.logps, *torch.autograd.grad(o.loss, leaves))
    if case["packed"]:
        out = _call("glu_packed")(t["gate_up"], activation=case["act"])
    else:
        out = _call("glu")(t["gate"], t["up"], activation=case["act"])
    return (out, *torch.autograd.grad(out, leaves, t["dout"]))


def _run_plain(case, t):
    with torch.no_grad():
        return {"qk": _plain_qk, "logps": _plain_logps, "preference": _plain_preference, "policy": _plain_policy,
                "glu": _plain_glu}[case["op"]](case, t)


def _plain_head(x, w, do, c, s, offset):
    """(normed and rotated x, its gradient and the weight's where the output's gradient `do` is given)."""
    half = c.shape[-1]
    f, w1 = x.float(), w.float() + offset
    r = torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
    n = f * r
    y = n * w1
    lo, hi = y[..., :half], y[..., half:]
    out = torch.cat([lo * c - hi * s, hi * c + lo * s], -1).to(x.dtype)
    if do is None:
        return out, None, None
    lo, hi = do.float()[..., :half], do.float()[..., half:]
    dy = torch.cat([lo * c + hi * s, hi * c - lo * s], -1)
    dw = (dy * n).sum((0, 1, 2), dtype=torch.float64).to(w.dtype)
    dn = dy * w1
    return out, (r * (dn - n * (dn * n).mean(-1, keepdim=True))).to(x.dtype), dw


def _plain_qk(case, t):
    cos, sin = t["cos"], t["sin"]
    if "positions" in t:
        cos, sin = cos[0][t["positions"]], sin[0][t["positions"]]
    half = case["head_dim"] // 2
    c, s = cos[..., :half].float().unsqueeze(1), sin[..., :half].float().unsqueeze(1)
    q, dq, dqw = _plain_head(t["q"], t["q_weight"], t.get("dq"), c, s, case["offset"])
    k, dk, dkw = _plain_head(t["k"], t["k_weight"], t.get("dk"), c, s, case["offset"])
    return (q, k, dq, dk, dqw, dkw) if case["train"] else (q, k)


def _plain_rows(logits, target, temperature):
    """(log-probabilities of the targets in 64 bits, probabilities in 32)."""
    z = logits.float()
    if temperature != 1.0:
        z = z / temperature
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    z_y = z.gather(-1, target.clamp(min=0).unsqueeze(-1))
    logp = ((z_y - m).double() - total.log()).squeeze(-1)
    return logp * (target != IGNORE), e.div_(total.float())


def _plain_dlogits(p, target, coef, dtype):
    """coef * (one at the target - p), zero where the target is ignored."""
    coef = (coef * (target != IGNORE)).float().unsqueeze(-1)
    return p.mul_(-coef).scatter_add_(-1, target.clamp(min=0).unsqueeze(-1), coef).to(dtype)


def _plain_logps(case, t):
    logp, p = _plain_rows(t["logits"], t["target"], case["temperature"])
    if not case["train"]:
        return (logp.float(),)
    return logp.float(), _plain_dlogits(p, t["target"], t["dlogps"] / case["temperature"], t["logits"].dtype)


def _plain_preference(case, t):
    beta, eps = 0.1, case["smoothing"]
    logp, p = _plain_rows(t["logits"], t["target"], 1.0)
    whole, share = logp.sum(-1), torch.ones_like(logp[:, 0])
    if case["normalized"]:
        share = 1.0 / (t["target"] != IGNORE).sum(-1).double()
        whole = whole * share
    over = whole - t["ref_logps"].double()
    pairs = over.numel() // 2
    diff = over[:pairs] - over[pairs:]
    h = beta * diff
    if case["kind"] == "sigmoid":
        up, down = torch.log1p(torch.exp(-h.abs())) + (-h).clamp(min=0), torch.log1p(torch.exp(-h.abs())) + h.clamp(min=0)
        loss, d = (1 - eps) * up + eps * down, beta * (eps - 1.0 + torch.sigmoid(h))
    else:
        loss, d = (diff - 0.5 / beta).square(), 2.0 * (diff - 0.5 / beta)
    coef = torch.cat([d, -d]) * share / pairs
    return (loss.mean().float(), whole.float(), (beta * over).float(),
            _plain_dlogits(p, t["target"], coef.unsqueeze(-1), t["logits"].dtype))


def _plain_policy(case, t):
    target, kl = t["target"], case["kl"]
    logp, p = _plain_rows(t["logits"], target, case["temperature"])
    kept = (target != IGNORE).double()
    adv = t["advantages"].double().unsqueeze(-1)
    ratio = torch.exp(logp - t["old_logps"].double()) if "old_logps" in t else torch.ones_like(logp)
    free, held = ratio * adv, ratio.clamp(0.8, 1.28) * adv
    loss, d = -torch.minimum(free, held), torch.where(free <= held, -free, torch.zeros_like(free))
    if kl:
        far = t["ref_logps"].double() - logp
        loss = loss + kl * (torch.expm1(far) - far)
        d = d - kl * torch.expm1(far)
    if case["reduction"] == "mean":
        weight = kept / kept.sum()
    elif case["reduction"] == "sequence":
        weight = kept / kept.sum(-1, keepdim=True) / kept.shape[0]
    else:
        weight = kept
    return ((loss * weight).sum().float(), logp.float(),
            _plain_dlogits(p, target, d * weight / case["temperature"], t["logits"].dtype))


def _plain_kept(x):
    """What 8 bits keep of x: groups of 32 along a row share 2^e, the least with |x| <= 127 * 2^e in the group."""
    rows, cols = x.shape
    g = torch.nn.functional.pad(x.float(), (0, -cols % GROUP)).view(rows, -1, GROUP)
    m, e = torch.frexp(g.abs().amax(-1, keepdim=True))
    e = (e - 7 + (m > 127 / 128)).clamp(min=-126)
    up, down = ((127 + e) << 23).int().view(torch.float32), ((127 - e) << 23).int().view(torch.float32)
    return (torch.round(g * down) * up).view(rows, -1)[:, :cols]


def _plain_act(x, act):
    """An activation and its slope."""
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-x))
        return x * s, s * (1.0 + x * (1.0 - s))
    if act == "gelu_tanh":
        a = math.sqrt(2.0 / math.pi)
        th = torch.tanh(a * (x + 0.044715 * x * x * x))
        return 0.5 * x * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * x * (1.0 - th * th) * a * (1.0 + 3 * 0.044715 * x * x)
    cdf = 0.5 * (1.0 + torch.erf(x / math.sqrt(2.0)))
    return x * cdf, cdf + x * torch.exp(-0.5 * x * x) / math.sqrt(2.0 * math.pi)


def _plain_glu(case, t):
    gate, up = t["gate_up"].split(case["cols"], 1) if case["packed"] else (t["gate"], t["up"])
    out = (_plain_act(gate.float(), case["act"])[0] * up.float()).to(gate.dtype)
    g, u, do = _plain_kept(gate), _plain_kept(up), t["dout"].float()
    a, slope = _plain_act(g, case["act"])
    dgate, dup = (do * u * slope).to(gate.dtype), (do * a).to(gate.dtype)
    return (out, torch.cat([dgate, dup], 1)) if case["packed"] else (out, dgate, dup)


# ---------------------------------------------------------------------------
# the work of a pass, and its results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op, e = case["op"], BYTES[case["dtype"]]
    if op == "qk":  # x -> out; out's gradient and x -> x's gradient; half tables, weights and theirs
        n = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        rows = min(case["batch"], 4096) if case["positions"] and case["seq"] == 1 else case["seq"]
        side = rows * case["head_dim"] * e + 2 * case["head_dim"] * e
        return {"bytes": (5 if case["train"] else 2) * n * e + (2 if case["train"] else 1) * side,
                "flops": (26 if case["train"] else 8) * n}
    if op == "glu":  # gate, up -> out and both in 8 bits with their scales; out's gradient and those -> two gradients
        n, scales = case["rows"] * case["cols"], case["rows"] * -(-case["cols"] // GROUP)
        return {"bytes": 6 * n * e + 2 * 2 * (n + scales), "flops": 30 * n}
    rows, kept = case["seqs"] * case["seq"], sum(b - a for a, b in _answers(case))
    v = case["vocab"]
    train = case.get("train", True)  # logits of the answers are read, and every row's gradient is written
    return {"bytes": (kept + (rows if train else 0)) * v * e + 8 * rows + 4 * rows, "flops": (8 if train else 4) * kept * v}


def exact(case, seed):
    t = {n: v.double() if v.is_floating_point() else v for n, v in _inputs(case, seed).items()}
    leaves = [t[n].requires_grad_(True) for n in _trained(case)]
    op = case["op"]
    if op == "qk":
        return _exact_qk(case, t, leaves)
    if op == "glu":
        return _exact_glu(case, t)
    target = t["target"]
    z = t["logits"] / case.get("temperature", 1.0)
    logp = z.gather(-1, target.clamp(min=0).unsqueeze(-1)).squeeze(-1) - torch.logsumexp(z, -1)
    logp = torch.where(target == IGNORE, 0.0, logp)
    kept = target != IGNORE
    if op == "logps":
        return (logp.detach(), *torch.autograd.grad(logp, leaves, t["dlogps"])) if leaves else (logp,)
    if op == "preference":
        whole = logp.sum(-1)
        if case["normalized"]:
            whole = whole / kept.sum(-1)
        reward = 0.1 * (whole - t["ref_logps"])
        h = torch.sub(*reward.chunk(2))
        if case["kind"] == "sigmoid":
            f = torch.nn.functional.logsigmoid
            loss = (-(1 - case["smoothing"]) * f(h) - case["smoothing"] * f(-h)).mean()
        else:
            loss = (h / 0.1 - 1 / (2 * 0.1)).pow(2).mean()
        return (loss.detach(), whole.detach(), reward.detach(), *torch.autograd.grad(loss, leaves))
    old = t.get("old_logps", logp.detach())
    ratio, adv = (logp - old).exp(), t["advantages"].view(-1, 1)
    loss = -torch.min(ratio * adv, ratio.clamp(1 - 0.2, 1 + 0.28) * adv)
    if case["kl"]:
        loss = loss + case["kl"] * ((t["ref_logps"] - logp).exp() - (t["ref_logps"] - logp) - 1)
    loss = loss * kept
    loss = {"mean": lambda: loss.sum() / kept.sum(), "sum": lambda: loss.sum(),
            "sequence": lambda: (loss.sum(-1) / kept.sum(-1)).mean()}[case["reduction"]]()
    return (loss.detach(), logp.detach(), *torch.autograd.grad(loss, leaves))


def _exact_qk(case, t, leaves):
    cos, sin = ((x[:, t["positions"].flatten()].unflatten(1, t["positions"].shape).squeeze(0) if "positions" in t else x)
                .unsqueeze(1) for x in (t["cos"], t["sin"]))
    outs = []
    for n in ("q", "k"):
        x = t[n] / (t[n].pow(2).mean(-1, keepdim=True) + EPS).sqrt() * (t[n + "_weight"] + case["offset"])
        a, b = x.chunk(2, -1)
        outs.append(x * cos + torch.cat([-b, a], -1) * sin)
    if not case["train"]:
        return tuple(outs)
    return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, (t["dq"], t["dk"])))


def _exact_glu(case, t):
    gate, up = t["gate_up"].detach().chunk(2, 1) if case["packed"] else (t["gate"].detach(), t["up"].detach())
    F = torch.nn.functional
    act = {"silu": F.silu, "gelu_exact": F.gelu, "gelu_tanh": lambda x: F.gelu(x, approximate="tanh")}[case["act"]]

    def kept(x):
        rows, cols = x.shape
        x = F.pad(x, (0, -cols % GROUP)).unflatten(1, (-1, GROUP))
        step = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 127)).clamp(min=-126))
        return (torch.round(x / step) * step).flatten(1)[:, :cols]

    g, u = kept(gate).requires_grad_(True), kept(up).requires_grad_(True)
    grads = torch.autograd.grad(act(g) * u, (g, u), t["dout"])
    return (act(gate) * up, torch.cat(grads, 1)) if case["packed"] else (act(gate) * up, *grads)
