"""The operators between the projections of a decoder layer whose speed is measured.

Beside the projections, norms and losses of perf/cases.py and the operators of perf/operators.py a
layer runs attention over packed prompts of different lengths (a training step, a prompt, or one
token a sequence), the norm with the residual's addition before it, and, where the frozen weights
are kept in 8 bits, products in 8-bit integers with a scale for each token and each channel, whose
tokens the norm hands over in 8 bits.

Where `own` is false the operators run in their plain form, elementary operations in 32 bits (sums
over the tokens, and values next to a rounding's border, in 64); where it is true they run through
the framework.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-6


def _own():
    """The framework's entry points."""
    root = str(Path.cwd() / "kernel-pocs_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from forge.kernels.attention import forge_varlen_attention
    from forge.kernels.int8 import Int8Weight, int8_linear
    from forge.kernels.rmsnorm import add_rmsnorm, add_rmsnorm_int8

    return {"attention": forge_varlen_attention, "norm": add_rmsnorm, "norm8": add_rmsnorm_int8,
            "linear8": int8_linear, "weight8": Int8Weight}


_calls = {}


def _call(name):
    if not _calls:
        _calls.update(_own())
    return _calls[name]


def listed():
    return [
        # a serving step of a few short sequences: one token each against its keys
        {"name": "attention_token", "op": "attention", "seqs": 4, "tokens": 4, "past": 2000, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "causal": True, "packed": False, "lse": False, "train": False, "dtype": "bf16"},
        # a serving step of many long sequences
        {"name": "attention_step", "op": "attention", "seqs": 32, "tokens": 32, "past": 131072, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "causal": True, "packed": False, "lse": False, "train": False, "dtype": "bf16"},
        # prompts of 8 sequences packed without padding, q, k and v columns of one projection's output
        {"name": "attention_prompt", "op": "attention", "seqs": 8, "tokens": 16384, "past": 0, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "causal": True, "packed": True, "lse": True, "train": False, "dtype": "bf16"},
        # a packed training batch
        {"name": "attention_train", "op": "attention", "seqs": 8, "tokens": 16384, "past": 0, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "causal": True, "packed": True, "lse": False, "train": True, "dtype": "bf16"},
        # short ragged sequences of narrow heads, seven to a group
        {"name": "attention_odd_fp16", "op": "attention", "seqs": 13, "tokens": 3001, "past": 0, "heads": 14,
         "kv_heads": 2, "head_dim": 64, "causal": True, "packed": False, "lse": False, "train": True, "dtype": "fp16"},
        # the residual's addition and norm of a full training batch
        {"name": "norm_train", "op": "norm", "rows": 8192, "cols": 4096, "offset": 0.0, "train": True, "dtype": "bf16"},
        # the same of a short batch in fp32 of an odd width, weights stored as their difference from one
        {"name": "norm_odd_fp32", "op": "norm", "rows": 1003, "cols": 2305, "offset": 1.0, "train": True,
         "dtype": "fp32"},
        # the norm and the gate and up projections of one serving step
        {"name": "norm_linear8_step", "op": "norm8", "rows": 16, "cols": 4096, "outs": 28672, "offset": 0.0,
         "dtype": "bf16"},
        # the norm and a projection of a whole batch (a reference model's forward pass)
        {"name": "norm_linear8", "op": "norm8", "rows": 8192, "cols": 4096, "outs": 14336, "offset": 0.0,
         "dtype": "bf16"},
        # one sequence through a small projection
        {"name": "linear8_short", "op": "linear8", "rows": 100, "cols": 4096, "outs": 1024, "bias": False,
         "train": False, "dtype": "bf16"},
        # a down projection of frozen 8-bit weights in a training step
        {"name": "linear8_train", "op": "linear8", "rows": 8192, "cols": 14336, "outs": 4096, "bias": False,
         "train": True, "dtype": "bf16"},
        # odd sizes with a bias
        {"name": "linear8_odd_fp16", "op": "linear8", "rows": 333, "cols": 1003, "outs": 2017, "bias": True,
         "train": True, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm: as often odd as it comes."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


MOST_PAIRS = 20_000_000 * 32 * 128  # query-key pairs times heads and head size: the listed batch's
HEADS = [(32, 8, 128), (32, 8, 128), (16, 8, 128), (32, 32, 128), (14, 2, 64), (32, 8, 64), (16, 4, 96), (8, 4, 256)]


def _draw_attention(rng):
    kind = rng.choice(["train", "train", "prompt", "step", "step"])
    while True:
        heads, kv, dim = rng.choice(HEADS)
        case = {"op": "attention", "seqs": _log(rng, 1, 64), "past": 0, "heads": heads, "kv_heads": kv, "head_dim": dim,
                "causal": kind == "step" or rng.random() < 0.85, "packed": rng.random() < 0.5 and kind != "step",
                "lse": kind == "prompt", "train": kind == "train", "dtype": rng.choice(["bf16", "bf16", "fp16"])}
        if kind == "step":
            case["tokens"], case["past"] = case["seqs"], _log(rng, 100, 150000)
        else:
            case["tokens"] = _log(rng, 64, 16384)
            if kind == "prompt" and rng.random() < 0.4:  # prompts that continue earlier tokens
                case["past"] = _log(rng, 100, 16384)
        if _pairs(case) * heads * dim <= MOST_PAIRS:
            return case


def draw(rng):
    op = rng.choice(["attention", "attention", "norm", "norm8", "linear8", "linear8"])
    if op == "attention":
        return _draw_attention(rng)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    offset = rng.choice([0.0, 0.0, 1.0])
    if op == "norm":
        cols = rng.choice([2048, 2560, 4096, 5120, 8192, _log(rng, 500, 10000)])
        train = rng.random() < 0.7
        most = 8192 * 4096 * 2 // (cols * BYTES[dtype])
        return {"op": op, "rows": _log(rng, 16 if train else 1, min(16384, most)), "cols": cols, "offset": offset,
                "train": train, "dtype": dtype}
    while True:
        cols = rng.choice([2048, 4096, 8192, 11008, 14336, _log(rng, 500, 14336)])
        outs = rng.choice([1024, 2560, 4096, 6144, 11008, 14336, _log(rng, 500, 16000)])
        case = {"op": op, "rows": _log(rng, 1, 8192), "cols": cols, "outs": outs, "dtype": dtype}
        if case["rows"] * cols * outs <= 8192 * 4096 * 14336:
            break
    if op == "norm8":
        return {**case, "offset": offset}
    return {**case, "bias": rng.random() < 0.3, "train": case["rows"] >= 16 and rng.random() < 0.5}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(n, total):
    """n whole numbers from about a quarter to almost twice the mean, that add up to total."""
    share = [0.3 + (0.381966 + 0.618034 * i) % 1.0 * 1.4 for i in range(n)]
    ends = [round(total * sum(share[:i + 1]) / sum(share)) for i in range(n)]
    return [b - a for a, b in zip([0] + ends, ends)]


def _spans(case):
    """(queries, keys) of each sequence: a step has one query each, a prompt its tokens after those before it."""
    n = case["seqs"]
    queries = [1] * n if case["tokens"] == n else _lengths(n, case["tokens"])
    return [(a, a + b) for a, b in zip(queries, _lengths(n, case["past"]))]


def _pairs(case):
    """Query-key pairs that the mask leaves."""
    if not case["causal"]:
        return sum(a * b for a, b in _spans(case))
    return sum(a * (b - a) + a * (a + 1) // 2 for a, b in _spans(case))


class _Draws:
    """Seeded tensors on the GPU."""

    def __init__(self, case, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = DTYPES[case["dtype"]]

    def normal(self, *shape, std=1.0, dtype=None):
        t = torch.empty(shape, dtype=dtype or self.dtype, device="cuda")
        return t.normal_(0.0, std, generator=self.g)


def _attention_inputs(case, seed):
    d = _Draws(case, seed)
    h, kv, dim = case["heads"], case["kv_heads"], case["head_dim"]
    spans = _spans(case)
    tokens, keys = (sum(x) for x in zip(*spans))
    if case["packed"] and tokens == keys:  # columns of one [T, (heads + 2 kv_heads) * head_dim] projection
        q, k, v = d.normal(tokens, h + 2 * kv, dim).split([h, kv, kv], 1)
    else:
        q, k, v = d.normal(tokens, h, dim), d.normal(keys, kv, dim), d.normal(keys, kv, dim)
    cu = torch.tensor([(0, 0)] + spans, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    t = {"q": q, "k": k, "v": v, "cu_q": cu[:, 0].contiguous(), "cu_k": cu[:, 1].contiguous()}
    if case["train"]:
        t["dout"] = d.normal(tokens, h, dim)
    return t


def _norm_inputs(case, seed):
    d = _Draws(case, seed)
    rows, cols = case["rows"], case["cols"]
    # the residual stream has grown over the layers before
    t = {"x": d.normal(rows, cols), "residual": d.normal(rows, cols, std=3.0),
         "weight": d.normal(cols, std=0.1).add_(1.0 - case["offset"])}
    if case.get("train"):  # the gradients of the normed rows and of the residual stream
        t["dy"], t["dh"] = d.normal(rows, cols), d.normal(rows, cols)
    if case["op"] == "norm8":
        t.update(_weight8(d, case["outs"], cols))
    return t


def _weight8(d, outs, cols):
    """A frozen weight of 8-bit integers, the largest of each channel 127, and its channels' scales."""
    w = d.normal(outs, cols, std=0.02, dtype=torch.float32)
    scale = w.abs().amax(1) / 127
    return {"qweight": torch.round(w / scale.unsqueeze(1)).to(torch.int8), "wscale": scale}


def _linear_inputs(case, seed):
    d = _Draws(case, seed)
    t = {"x": d.normal(case["rows"], case["cols"]), **_weight8(d, case["outs"], case["cols"])}
    if case["bias"]:
        t["bias"] = d.normal(case["outs"])
    if case["train"]:
        t["dy"] = d.normal(case["rows"], case["outs"])
    return t


def _inputs(case, seed):
    return {"attention": _attention_inputs, "linear8": _linear_inputs}.get(case["op"], _norm_inputs)(case, seed)


def _trained(case):
    """The names of the inputs whose gradients the pass returns."""
    if not case.get("train"):
        return []
    return {"attention": ["q", "k", "v"], "norm": ["x", "residual", "weight"], "linear8": ["x"]}[case["op"]]


def prepare(case, seed):
    t = _inputs(case, seed)
    for n in _trained(case):
        t[n] = t[n].detach().requires_grad_(True)
    if own and "qweight" in t:  # the program lays its weights out once
        t["handle"] = _call("weight8")(t["qweight"], t["wscale"], backward=bool(case.get("train")))
    return case, t


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case, t = state
    return (_run_own if own else _run_plain)(case, t)


def _run_own(case, t):
    op, train = case["op"], case.get("train")
    leaves = [t[n] for n in _trained(case)]
    if op == "attention":
        out = _call("attention")(t["q"], t["k"], t["v"], t["cu_q"], t["cu_k"], causal=case["causal"],
                                 return_lse=case["lse"])
        if case["lse"]:
            return out
        return (out, *torch.autograd.grad(out, leaves, t["dout"])) if train else (out,)
    if op == "norm":
        y, h = _call("norm")(t["x"], t["residual"], t["weight"], eps=EPS, offset=case["offset"])
        return (y, h, *torch.autograd.grad((y, h), leaves, (t["dy"], t["dh"]))) if train else (y, h)
    if op == "norm8":
        rows, h = _call("norm8")(t["x"], t["residual"], t["weight"], eps=EPS, offset=case["offset"])
        return _call("linear8")(rows, t["handle"]), h
    y = _call("linear8")(t["x"], t["handle"], bias=t.get("bias"))
    return (y, *torch.autograd.grad(y, leaves, t["dy"])) if train else (y,)


def _run_plain(case, t):
    with torch.no_grad():
        return {"attention": _plain_attention, "norm": _plain_norm, "norm8": _plain_norm8,
                "linear8": _plain_linear8}[case["op"]](case, t)


def _plain_attention(case, t):
    q, k, v, do = t["q"], t["k"], t["v"], t.get("dout")
    group, scale = case["heads"] // case["kv_heads"], case["head_dim"] ** -0.5
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    grads = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v)] if case["train"] else []

    def rows(x, at, heads):  # the rows of a sequence as [kv_heads, group * tokens, head_dim]
        x = x[at, heads].transpose(0, 1).float()
        return x.reshape(-1, group * x.shape[1], x.shape[2])

    def put(x, at, heads, value):
        x[at, heads] = value.reshape(-1, at.stop - at.start, value.shape[-1]).transpose(0, 1).to(x.dtype)

    a = b = 0
    for n_q, n_k in _spans(case):
        at_q, at_k = slice(a, a + n_q), slice(b, b + n_k)
        a, b = a + n_q, b + n_k
        if n_q == 0:
            continue
        hidden = None
        if case["causal"] and n_q > 1:
            keys = torch.arange(n_k, device=q.device)
            hidden = (keys > keys[n_k - n_q:].unsqueeze(1)).repeat(group, 1)
        step = max(1, min(case["kv_heads"], 2 ** 30 // (group * n_q * n_k)))  # heads whose scores fit beside each other
        for g in range(0, case["kv_heads"], step):
            at_kv = slice(g, min(g + step, case["kv_heads"]))
            at_h = slice(at_kv.start * group, at_kv.stop * group)
            qs, ks, vs = rows(q, at_q, at_h), k[at_k, at_kv].transpose(0, 1).float(), v[at_k, at_kv].transpose(0, 1).float()
            s = torch.matmul(qs, ks.transpose(1, 2)).mul_(scale)
            if hidden is not None:
                s.masked_fill_(hidden, -math.inf)
            m = s.amax(-1, keepdim=True)
            p = s.sub_(m).exp_()
            total = p.sum(-1, keepdim=True)
            p.div_(total)
            o = torch.matmul(p, vs)
            put(out, at_q, at_h, o)
            lse[at_q, at_h] = (m + total.log()).reshape(-1, n_q).t()
            if not case["train"]:
                continue
            dos = rows(do, at_q, at_h)
            grads[2][at_k, at_kv] = torch.matmul(p.transpose(1, 2), dos).transpose(0, 1).to(v.dtype)
            ds = torch.matmul(dos, vs.transpose(1, 2)).sub_((dos * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            put(grads[0], at_q, at_h, torch.matmul(ds, ks))
            grads[1][at_k, at_kv] = torch.matmul(ds.transpose(1, 2), qs).transpose(0, 1).to(k.dtype)
    return (out, lse) if case["lse"] else (out, *grads)


def _plain_norm(case, t):
    h = (t["x"].float() + t["residual"].float()).to(t["x"].dtype)
    f, w = h.float(), t["weight"].float() + case["offset"]
    r = torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
    n = f * r
    y = (n * w).to(h.dtype)
    if not case["train"]:
        return y, h
    dy = t["dy"].float()
    dn = dy * w
    d = (t["dh"].float() + r * (dn - n * (dn * n).mean(-1, keepdim=True))).to(h.dtype)
    return y, h, d, d, (dy * n).sum(0, dtype=torch.float64).to(t["weight"].dtype)


def _plain_quantize(t):
    """(whole numbers from -127 to 127 as floats, largest magnitudes) of the rows of 64-bit values."""
    a = t.abs().amax(-1, keepdim=True)
    return torch.round(127 * t / torch.where(a > 0, a, torch.ones_like(a))).float(), a


def _plain_product(q, w):
    """Sums of products of 8-bit integers: exact in 32 bits over 1024 products, added up in 64."""
    total = torch.zeros(q.shape[0], w.shape[0], dtype=torch.float64, device=q.device)
    for c in range(0, q.shape[1], 1024):
        total += torch.matmul(q[:, c:c + 1024], w[:, c:c + 1024].float().t())
    return total


def _plain_norm8(case, t):
    h = (t["x"].float() + t["residual"].float()).to(t["x"].dtype)
    r = torch.rsqrt(h.float().square().mean(-1, keepdim=True) + EPS)
    q, a = _plain_quantize(h.double() * (t["weight"].double() + case["offset"]))
    y = _plain_product(q, t["qweight"]) * (a.float() * r / 127) * t["wscale"]
    return y.to(h.dtype), h


def _plain_linear8(case, t):
    x, w = t["x"], t["qweight"]
    q, a = _plain_quantize(x.double())
    y = _plain_product(q, w) * (a.float() / 127) * t["wscale"]
    if case["bias"]:
        y = y + t["bias"]
    if not case["train"]:
        return (y.to(x.dtype),)
    q, a = _plain_quantize(t["dy"].double() * t["wscale"])
    return y.to(x.dtype), (_plain_product(q, w.t()) * (a.float() / 127)).to(x.dtype)


# ---------------------------------------------------------------------------
# the work of a pass, and its results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op, e = case["op"], BYTES[case["dtype"]]
    if op == "attention":  # q, k, v -> out (and out's gradient and those -> three gradients)
        tokens, keys = (sum(x) for x in zip(*_spans(case)))
        q, kv = tokens * case["heads"] * case["head_dim"] * e, keys * case["kv_heads"] * case["head_dim"] * e
        both = (5 * q + 6 * kv) if case["train"] else 2 * q + 2 * kv
        return {"bytes": both, "flops": (14 if case["train"] else 4) * _pairs(case) * case["heads"] * case["head_dim"]}
    rows, cols = case["rows"], case["cols"]
    if op == "norm":  # x, residual -> y, h; dy, dh, h -> d
        n = rows * cols
        return {"bytes": (8 if case["train"] else 4) * n * e + 2 * cols * e, "flops": (18 if case["train"] else 6) * n}
    outs, passes = case["outs"], 2 if case.get("train") else 1
    if op == "norm8":  # x, residual, 8-bit weights -> h, y
        return {"bytes": 3 * rows * cols * e + outs * cols + rows * outs * e, "flops": 2 * rows * cols * outs}
    return {"bytes": passes * ((rows * cols + rows * outs) * e + outs * cols), "flops": passes * 2 * rows * cols * outs}


def exact(case, seed):
    op = case["op"]
    t = {n: v.double() if v.is_floating_point() else v for n, v in _inputs(case, seed).items()}
    if op == "attention":
        return _exact_attention(case, t)
    leaves = [t[n].requires_grad_(True) for n in _trained(case)]
    if op == "linear8":
        return _exact_linear8(case, t)
    dtype = DTYPES[case["dtype"]]
    stored = (t["x"] + t["residual"]).detach().to(dtype).double()  # the stream is stored in its type, and normed as stored
    h = t["x"] + t["residual"]
    h = h + (stored - h).detach()
    w = t["weight"] + case["offset"]
    rms = (h.pow(2).sum(-1, keepdim=True) / h.shape[1] + EPS).sqrt()
    if op == "norm8":
        q, unit = _exact_rows(h * w)
        return q @ t["qweight"].double().T * (unit / rms) * t["wscale"], h
    y = h / rms * w
    if not leaves:
        return y, h
    return (y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (t["dy"], t["dh"])))


def _exact_rows(t):
    """(whole numbers, the value of one) of each row."""
    top = t.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, t * 127 / top, t).round(), top / 127


def _exact_linear8(case, t):
    w = t["qweight"].double()
    q, unit = _exact_rows(t["x"].detach())
    y = unit * torch.nn.functional.linear(q, w) * t["wscale"]
    if case["bias"]:
        y += t["bias"]
    if not case["train"]:
        return (y,)
    q, unit = _exact_rows(t["dy"] * t["wscale"])
    return y, unit * (q @ w)


def _exact_attention(case, t):
    h, kv, dim = case["heads"], case["kv_heads"], case["head_dim"]
    parts, lses = [], []
    grads = [torch.zeros_like(t[n]) for n in ("q", "k", "v")] if case["train"] else []
    cu_q, cu_k = t["cu_q"].tolist(), t["cu_k"].tolist()
    for i in range(case["seqs"]):
        rows, cols = slice(*cu_q[i:i + 2]), slice(*cu_k[i:i + 2])
        n_q, n_k = rows.stop - rows.start, cols.stop - cols.start
        if n_q == 0:
            continue
        allowed = torch.ones(n_q, n_k, dtype=torch.bool, device="cuda")
        if case["causal"]:
            allowed = allowed.tril(n_k - n_q)
        outs, sums = [], []
        for j in range(h):
            q, k, v = (t[n][r, c].detach().requires_grad_(case["train"])
                       for n, r, c in (("q", rows, j), ("k", cols, j * kv // h), ("v", cols, j * kv // h)))
            score = (q @ k.T / math.sqrt(dim)).where(allowed, -math.inf)
            out = score.softmax(-1) @ v
            if case["train"]:
                for total, c, part in zip(grads, (j, j * kv // h, j * kv // h),
                                          torch.autograd.grad(out, (q, k, v), t["dout"][rows, j])):
                    total[rows if total is grads[0] else cols, c] += part
            outs.append(out.detach())
            sums.append(score.detach().logsumexp(-1))
        parts.append(torch.stack(outs, 1))
        lses.append(torch.stack(sums, 1))
    return (torch.cat(parts), torch.cat(lses)) if case["lse"] else (torch.cat(parts), *grads)
