"""The operators of a preference or policy fine-tuning step, run as they are
used: through the patch adapters' options, and together in one step of a small
decoder layer with its loss, against the same step in float64."""
import copy
import math

import pytest
import torch
import torch.nn as nn

from oracle import glu_act8 as OG
from oracle import logprob as OL
from oracle.qk_norm_rope import forward as qk_forward

IGNORE = -100


def _cos_sin(rows, dim, dtype, device):
    inv = 1.0 / 10000.0 ** (torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    ang = torch.arange(rows, dtype=torch.float64).unsqueeze(1) * inv
    ang = torch.cat([ang, ang], 1)
    return tuple(t.to(device=device, dtype=dtype).unsqueeze(0) for t in (ang.cos(), ang.sin()))


# ---------------------------------------------------------------------------
# patch adapters
# ---------------------------------------------------------------------------
def test_saved_activations_option():
    from forge.patching import FORWARD_MAKERS

    class MLP(nn.Module):
        def __init__(self, act):
            super().__init__()
            self.gate_proj, self.up_proj, self.down_proj = nn.Linear(8, 12), nn.Linear(8, 12), nn.Linear(12, 8)
            self.config = type("C", (), {"hidden_act": act})()

    x = torch.randn(3, 8)
    for kernel, act in (("swiglu", "silu"), ("geglu", "gelu"), ("geglu", "gelu_pytorch_tanh")):
        m = MLP(act)
        with pytest.raises(ValueError, match="saved_activations"):
            FORWARD_MAKERS[kernel](m, {"saved_activations": "4bit"})
        # a CPU call takes the path without the option
        assert torch.equal(FORWARD_MAKERS[kernel](m, {"saved_activations": "8bit"})(x), FORWARD_MAKERS[kernel](m, {})(x))


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,act,kind", [("swiglu", "silu", "silu"), ("geglu", "gelu", "gelu_exact"),
                                             ("geglu", "gelu_pytorch_tanh", "gelu_tanh")])
def test_saved_activations_in_8_bits(kernel, act, kind):
    from forge.kernels.glu_act8 import glu_act8
    from forge.patching import FORWARD_MAKERS

    class MLP(nn.Module):
        def __init__(self):
            super().__init__()
            kw = {"device": "cuda", "dtype": torch.bfloat16}
            self.gate_proj, self.up_proj = nn.Linear(256, 688, **kw), nn.Linear(256, 688, **kw)
            self.down_proj = nn.Linear(688, 256, **kw)
            self.config = type("C", (), {"hidden_act": act})()

    torch.manual_seed(0)
    m = MLP()
    x = torch.randn(2, 37, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    forward = FORWARD_MAKERS[kernel](m, {"saved_activations": "8bit"})
    out = forward(x)
    want = m.down_proj(glu_act8(m.gate_proj(x), m.up_proj(x), kind))
    assert torch.equal(out, want)
    g = torch.randn_like(out)
    got = torch.autograd.grad(out, [x, m.gate_proj.weight, m.up_proj.weight], g)
    plain = torch.autograd.grad(FORWARD_MAKERS[kernel](m, {})(x), [x, m.gate_proj.weight, m.up_proj.weight], g)
    for a, b in zip(got, plain):  # half a step of 1/127 of a group's largest: about 0.3% of a value's deviation
        assert (a.float() - b.float()).norm() <= 2e-2 * b.float().norm()


@pytest.mark.gpu
@pytest.mark.parametrize("cos_batch", [1, 2])
def test_fused_qk_norm_of_a_patched_attention(cos_batch):
    """A LoRA attention with q/k norms, patched with and without the option,
    next to an fp32 copy: the one-pass errors may not exceed twice the modules'
    or 1% of the scale (what the adapters' own tests allow)."""
    pytest.importorskip("transformers")
    from test_patch_adapters import _check, _run, build

    from forge.patching import FORWARD_MAKERS
    from forge.patching.kernels.lora import qk_norm_args

    m, rot = build("qwen3", "attn", dtype=torch.bfloat16, device="cuda")
    with torch.no_grad():
        m.q_norm.weight.normal_(1.0, 0.2)
        m.k_norm.weight.normal_(1.0, 0.2)
    m32, plain = copy.deepcopy(m).float(), copy.deepcopy(m)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, 37, 512, device="cuda", generator=g)
    cos, sin = rot(x, torch.arange(37, device="cuda")[None].expand(cos_batch, 37))
    dy = torch.randn(2, 37, 512, device="cuda", generator=g)
    bf = torch.bfloat16
    r32 = _run(m32, x, ((cos.float(), sin.float()), None), "attn", dy)
    plain.forward = FORWARD_MAKERS["lora_qkv"](plain, {})
    rp = _run(plain, x.to(bf), ((cos.to(bf), sin.to(bf)), None), "attn", dy)
    m.forward = FORWARD_MAKERS["lora_qkv"](m, {"fuse_qk_norm": True})
    rf = _run(m, x.to(bf), ((cos.to(bf), sin.to(bf)), None), "attn", dy)
    _check(rf[0], rp[0], r32[0], "out")
    _check(rf[1], rp[1], r32[1], "dx")
    for i, (a, b, c) in enumerate(zip(rf[2], rp[2], r32[2])):
        _check(a, b, c, f"lora grad {i}")
    for name in ("q_norm", "k_norm"):
        a, b, c = (getattr(t, name).weight.grad for t in (m, plain, m32))
        _check(a, b, c, name)
    Q, K = torch.zeros(2, 37, 4, 128, device="cuda", dtype=bf), torch.zeros(2, 37, 2, 128, device="cuda", dtype=bf)
    c16, s16 = cos.to(bf), sin.to(bf)
    assert qk_norm_args(m, Q, K, c16, s16, {})[3] == 0.0
    assert qk_norm_args(m, Q, K, c16, s16, {"qk_norm_offset": 1.0})[3] == 1.0
    # what the one pass does not take goes to the modules
    assert qk_norm_args(m, Q, K, c16[..., :64], s16[..., :64], {}) is None
    assert qk_norm_args(m, Q.cpu(), K.cpu(), c16, s16, {}) is None
    handle = m.q_norm.register_forward_hook(lambda *a: None)
    assert qk_norm_args(m, Q, K, c16, s16, {}) is None
    handle.remove()
    m.k_norm.variance_epsilon = 1e-3
    assert qk_norm_args(m, Q, K, c16, s16, {}) is None


class GemmaToyRMSNorm(nn.Module):
    def __init__(self):
        super().__init__()
        self.eps, self.weight = 1e-6, nn.Parameter(torch.zeros(8))


class _Normed(nn.Module):
    def __init__(self):
        super().__init__()
        self.q_norm, self.k_norm = GemmaToyRMSNorm(), GemmaToyRMSNorm()


def test_qk_norm_args_without_norms_or_on_the_cpu():
    from forge.patching.kernels.lora import qk_norm_args

    Q, table = torch.zeros(1, 3, 2, 8), torch.zeros(1, 3, 8)
    assert qk_norm_args(_Normed(), Q, Q, table, table, {}) is None
    assert qk_norm_args(nn.Linear(2, 2), Q, Q, table, table, {}) is None


@pytest.mark.gpu
def test_qk_norm_offset_by_class():
    from forge.patching.kernels.lora import qk_norm_args

    Q, table = torch.zeros(1, 3, 2, 8, device="cuda"), torch.zeros(1, 3, 8, device="cuda")
    m = _Normed().cuda()
    assert qk_norm_args(m, Q, Q, table, table, {})[2:] == (1e-6, 1.0)
    assert qk_norm_args(m, Q, Q, table, table, {"qk_norm_offset": 0.0})[3] == 0.0


# ---------------------------------------------------------------------------
# one step
# ---------------------------------------------------------------------------
H, NQ, NK, D, I, V, N, S = 64, 4, 2, 16, 96, 301, 4, 24
NAMES = ["embed", "qkv", "qn", "kn", "o", "gate_up", "down", "head"]


def _params(seed):
    g = torch.Generator().manual_seed(seed)
    shapes = {"embed": (V, H), "qkv": ((NQ + 2 * NK) * D, H), "qn": (D,), "kn": (D,), "o": (H, NQ * D),
              "gate_up": (2 * I, H), "down": (H, I), "head": (V, H)}
    p = {n: torch.randn(*s, generator=g, dtype=torch.float64) / math.sqrt(s[-1]) for n, s in shapes.items()}
    p["qn"], p["kn"] = 1 + 0.2 * p["qn"] * 4, 1 + 0.2 * p["kn"] * 4
    p["head"] *= 3.0
    return p


def _attention(q, k, v):
    """Causal attention of [B, heads, S, D] in q's dtype's own products."""
    k, v = k.repeat_interleave(NQ // NK, 1), v.repeat_interleave(NQ // NK, 1)
    a = (q.float() if q.dtype != torch.float64 else q) @ k.to(q.dtype if q.dtype == torch.float64 else torch.float32).mT
    a = a / math.sqrt(D)
    a = a.masked_fill(torch.ones(S, S, dtype=torch.bool, device=q.device).triu(1), float("-inf")).softmax(-1)
    return (a @ v.to(a.dtype)).to(q.dtype)


def _decoder(p, ids, norm, qk, glu):
    x = p["embed"][ids]
    qkv = (norm(x) @ p["qkv"].T).view(N, S, NQ + 2 * NK, D)
    q, k, v = (t.transpose(1, 2) for t in qkv.split([NQ, NK, NK], 2))
    q, k = qk(q, k)
    x = x + _attention(q, k, v).transpose(1, 2).reshape(N, S, NQ * D) @ p["o"].T
    x = x + glu(norm(x) @ p["gate_up"].T) @ p["down"].T
    return norm(x) @ p["head"].T


class _PlainGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate_up):
        gate, up = gate_up.reshape(-1, 2 * I).chunk(2, -1)
        ctx.save_for_backward(OG.kept(gate.float()), OG.kept(up.float()))
        ctx.shape = gate_up.shape
        return (OG.act_and_slope(gate, "silu")[0] * up).view(*gate_up.shape[:-1], I)

    @staticmethod
    def backward(ctx, dout):
        g, u = ctx.saved_tensors
        d = dout.reshape(-1, I)
        act, slope = OG.act_and_slope(g, "silu")
        return torch.cat([d * u * slope, d * act], -1).view(ctx.shape)


def _batch():
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, V, (N, S), generator=g)
    target = torch.full((N, S), IGNORE)
    target[:, :-1] = ids[:, 1:]  # the next token, with the logits left whole
    for i, (a, b) in enumerate([(3, 24), (5, 20), (0, 24), (10, 11)]):
        target[i, :a] = IGNORE
        target[i, b:] = IGNORE
    return ids, target


@pytest.mark.gpu
@pytest.mark.parametrize("loss", ["policy", "preference"])
@pytest.mark.parametrize("dtype,most", [(torch.float32, 1e-3), (torch.bfloat16, 6e-2)], ids=str)
def test_one_step_against_float64(dtype, most, loss):
    """Gradients of every weight.  fp32: gate and up differ from the float64
    step's by about 1e-5 of a group's largest, so 2 * 127 * 1e-5 of the kept
    values round to the other neighbour, 1/127 away: sqrt(2.5e-3) / 127 = 4e-4
    of a gradient's norm.  bf16: rounding of 2^-9 at some 40 places."""
    from forge.kernels.glu_act8 import glu_act8_packed
    from forge.kernels.logprob import forge_policy_loss, forge_preference_loss, forge_token_logps
    from forge.kernels.rmsnorm import apply_rmsnorm
    from forge.kernels.rope import apply_qk_norm_rope

    ids, target = _batch()
    p64 = {n: t.to(dtype).double().requires_grad_(True) for n, t in _params(0).items()}
    ref64 = {n: t.to(dtype).double() for n, t in _params(0).items()}
    g = torch.Generator().manual_seed(9)
    for n in ("head", "down"):
        ref64[n] = (ref64[n] + 0.02 * torch.randn(ref64[n].shape, generator=g)).to(dtype).double()
    p = {n: t.detach().to("cuda", dtype).requires_grad_(True) for n, t in p64.items()}
    ref = {n: t.to("cuda", dtype) for n, t in ref64.items()}
    adv = torch.tensor([1.0, -0.5, 0.7, -1.2])
    cos, sin = _cos_sin(S, D, torch.float64, "cpu")
    cosg, sing = _cos_sin(S, D, torch.float32, "cuda")
    ones = torch.ones(H, device="cuda", dtype=dtype)

    def norm64(x):
        return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()

    def logits64(q):
        c, s = cos[..., :D // 2].unsqueeze(1), sin[..., :D // 2].unsqueeze(1)
        return _decoder(q, ids, norm64, lambda a, b: (qk_forward(a, q["qn"], c, s, 1e-6, 0.0),
                                                      qk_forward(b, q["kn"], c, s, 1e-6, 0.0)), _PlainGLU.apply)

    def logits_own(q):
        return _decoder(q, ids.cuda(), lambda x: apply_rmsnorm(x, ones, eps=1e-6, in_place=False),
                        lambda a, b: apply_qk_norm_rope(a, b, q["qn"], q["kn"], cosg, sing), glu_act8_packed)

    kept = target != IGNORE
    with torch.no_grad():
        lp_ref = OL.token_logps(logits64(ref64), target)
        own_ref = forge_token_logps(logits_own(ref), target.cuda())
    lp = OL.token_logps(logits64(p64), target)
    own = logits_own(p)
    if loss == "policy":
        ratio, a = (lp - lp_ref).exp(), adv.unsqueeze(1)
        each = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a) + 0.1 * (torch.expm1(lp_ref - lp) - (lp_ref - lp))
        want = (torch.where(kept, each, 0.0).sum(-1) / kept.sum(-1)).mean()
        o = forge_policy_loss(own, target.cuda(), adv.cuda(), own_ref, own_ref, kl_coef=0.1, reduction="sequence")
    else:
        c, r = ((lp - lp_ref) * kept).sum(-1).chunk(2)
        want = -torch.nn.functional.logsigmoid(0.5 * (c - r)).mean()
        o = forge_preference_loss(own, target.cuda(), own_ref.sum(-1), beta=0.5)
    want_grads = torch.autograd.grad(want, [p64[n] for n in NAMES])
    got_grads = torch.autograd.grad(o.loss, [p[n] for n in NAMES])
    assert abs(o.loss.item() - want.item()) <= most * (abs(want.item()) + 0.1)
    for n, a, b in zip(NAMES, got_grads, want_grads):
        off = (a.double().cpu() - b).norm() / b.norm()
        assert off <= most, (n, off.item())


@pytest.mark.gpu
def test_serving_steps_agree_with_the_whole_sequence():
    """Queries and keys of a sequence a token at a time, and the tokens'
    log-probabilities, against one call over the sequence."""
    from forge.kernels.logprob import forge_token_logps
    from forge.kernels.rope import apply_qk_norm_rope

    torch.manual_seed(0)
    b, s, d, v = 3, 12, 128, 20011
    q = torch.randn(b, s, 8, d, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    k = torch.randn(b, s, 2, d, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    qw, kw = torch.rand(2, d, device="cuda", dtype=torch.bfloat16) + 0.5
    cos, sin = _cos_sin(64, d, torch.bfloat16, "cuda")
    start = torch.tensor([[0], [7], [40]], device="cuda")
    whole = apply_qk_norm_rope(q, k, qw, kw, cos, sin, start + torch.arange(s, device="cuda"))
    logits = torch.randn(b, s, v, device="cuda", dtype=torch.bfloat16)
    target = torch.randint(0, v, (b, s), device="cuda")
    scores = forge_token_logps(logits, target)
    for i in range(s):
        step = apply_qk_norm_rope(q[:, :, i:i + 1], k[:, :, i:i + 1], qw, kw, cos, sin, start + i)
        assert all(torch.equal(a, w[:, :, i:i + 1]) for a, w in zip(step, whole))
        one = forge_token_logps(logits[:, i], target[:, i])
        assert (one - scores[:, i]).abs().max() <= 2 * (64 + 3 + 3 * 14) * 2.0 ** -24
