"""What the fused q/k norm + RoPE of a patched attention takes from the model:
the weight's offset and the rotation, each read from the module's own forward
and not from a name."""
import importlib

import pytest
import torch
import torch.nn as nn

transformers = pytest.importorskip("transformers")

# (modeling module, norm class of its q and k heads, offset its forward adds to the weight)
NORMS = [("qwen3", "Qwen3RMSNorm", 0.0), ("qwen3_moe", "Qwen3MoeRMSNorm", 0.0), ("qwen3_next", "Qwen3NextRMSNorm", 1.0),
         ("gemma2", "Gemma2RMSNorm", 1.0), ("gemma3", "Gemma3RMSNorm", 1.0), ("gemma3n", "Gemma3nRMSNorm", 0.0),
         ("gemma4", "Gemma4RMSNorm", 0.0), ("t5gemma2", "T5Gemma2RMSNorm", 1.0),
         ("minimax_m3_vl", "MiniMaxM3VLRMSNorm", 1.0), ("apertus", "ApertusRMSNorm", 0.0),
         ("dots1", "Dots1RMSNorm", 0.0), ("llama", "LlamaRMSNorm", 0.0)]


def _class(model, name):
    try:
        module = importlib.import_module(f"transformers.models.{model}.modeling_{model}")
    except ImportError:
        pytest.skip(f"transformers {transformers.__version__} has no {model}")
    return getattr(module, name)


def _eps(norm):
    return getattr(norm, "variance_epsilon", getattr(norm, "eps", None))


@pytest.mark.parametrize("model,name,offset", NORMS)
def test_offset_of_each_norm(model, name, offset):
    from forge.patching.kernels.lora import norm_offset

    norm = _class(model, name)(24, eps=1e-3)
    g = torch.Generator().manual_seed(0)
    with torch.no_grad():
        norm.weight.copy_(torch.randn(24, generator=g))
    assert norm_offset(norm, _eps(norm)) == offset
    x = torch.randn(5, 24, generator=g) * 0.05
    want = x * (x.square().mean(-1, keepdim=True) + 1e-3).rsqrt() * (norm.weight + offset)
    torch.testing.assert_close(norm(x), want, rtol=1e-5, atol=1e-6)  # fp32: some 10 roundings
    assert norm_offset(norm, 1e-6) is None  # an eps that is not the one it uses


class _Base(nn.Module):
    def __init__(self, dim=24):
        super().__init__()
        self.eps, self.weight = 1e-6, nn.Parameter(torch.ones(dim))

    def normed(self, x):
        return x * (x.square().mean(-1, keepdim=True) + self.eps).rsqrt()


class HalfRMSNorm(_Base):  # neither offset
    def forward(self, x):
        return self.normed(x) * (0.5 + self.weight)


class ShiftedRMSNorm(_Base):  # a bias besides
    def __init__(self):
        super().__init__()
        self.bias = nn.Parameter(torch.zeros(24))

    def forward(self, x):
        return self.normed(x) * self.weight + self.bias


class GatedRMSNorm(_Base):  # takes another input
    def forward(self, x, gate):
        return self.normed(x) * self.weight * gate


class FlaggedRMSNorm(_Base):  # its attribute says which
    def __init__(self, plus_one):
        super().__init__()
        self.plus_one = plus_one

    def forward(self, x):
        return self.normed(x) * (self.weight + 1.0 if self.plus_one else self.weight)


def test_norms_that_are_something_else():
    from forge.patching import FORWARD_MAKERS
    from forge.patching.kernels.lora import norm_offset

    assert all(norm_offset(n, 1e-6) is None for n in (HalfRMSNorm(), ShiftedRMSNorm(), GatedRMSNorm()))
    assert norm_offset(FlaggedRMSNorm(True), 1e-6) == 1.0 and norm_offset(FlaggedRMSNorm(False), 1e-6) == 0.0
    flagged = FlaggedRMSNorm(False)
    flagged.plus_one = True
    assert norm_offset(flagged, 1e-6) == 1.0
    flagged.eps = 0.0
    assert norm_offset(flagged, 0.0) == 1.0 and norm_offset(flagged, 1e-6) is None
    # a forward of the instance's own: only the framework's adapter of the same norm is known
    patched = FlaggedRMSNorm(False)
    patched.forward = lambda x: x
    assert norm_offset(patched, 1e-6) is None
    patched.forward = FORWARD_MAKERS["rmsnorm"](patched, {})
    assert norm_offset(patched, 1e-6) == 0.0
    # weights that are not what they were, on whatever device, are not looked at
    meta = FlaggedRMSNorm(True).to("meta")
    assert norm_offset(meta, 1e-6) == 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("model,name,offset", [n for n in NORMS if n[0] in (
    "gemma3", "gemma3n", "gemma4", "t5gemma2", "minimax_m3_vl", "qwen3_next")])
def test_fused_attention_with_the_norms_of_other_models(model, name, offset, monkeypatch):
    """A patched attention whose norms are another model's class, with the
    option and without, beside an fp32 copy."""
    import copy

    from test_patch_adapters import _check, _run, build

    from forge.patching import FORWARD_MAKERS

    import forge.kernels.rope  # noqa: F401  (takes the name before it is replaced)
    import kernels.rope.qk_norm_rope as qk

    calls, apply = [], qk.apply_qk_norm_rope
    monkeypatch.setattr(qk, "apply_qk_norm_rope", lambda *a, **k: (calls.append(k["offset"]), apply(*a, **k))[1])
    m, rot = build("qwen3", "attn", dtype=torch.bfloat16, device="cuda")
    torch.manual_seed(3)
    for n in ("q_norm", "k_norm"):
        norm = _class(model, name)(128, eps=1e-6).to("cuda", torch.bfloat16)
        with torch.no_grad():
            norm.weight.normal_(1.0 - offset, 0.2)
        setattr(m, n, norm)
    m32, plain = copy.deepcopy(m).float(), copy.deepcopy(m)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(2, 37, 512, device="cuda", generator=g) for _ in range(2))
    cos, sin = rot(x, torch.arange(37, device="cuda")[None])
    bf = torch.bfloat16
    r32 = _run(m32, x, ((cos.float(), sin.float()), None), "attn", dy)
    plain.forward = FORWARD_MAKERS["lora_qkv"](plain, {})
    m.forward = FORWARD_MAKERS["lora_qkv"](m, {"fuse_qk_norm": True})
    rp, rf = (_run(t, x.to(bf), ((cos.to(bf), sin.to(bf)), None), "attn", dy) for t in (plain, m))
    assert calls == [offset]
    _check(rf[0], rp[0], r32[0], "out")
    _check(rf[1], rp[1], r32[1], "dx")
    for n in ("q_norm", "k_norm"):
        a, b, c = (getattr(t, n).weight.grad for t in (m, plain, m32))
        _check(a, b, c, n)


def test_hooks_of_a_norm():
    from forge.patching.kernels.lora import has_hooks

    for register in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook",
                     "register_full_backward_pre_hook"):
        norm = FlaggedRMSNorm(False)
        assert not has_hooks(norm)
        handle = getattr(norm, register)(lambda *a: None)
        assert has_hooks(norm), register
        handle.remove()
        assert not has_hooks(norm)
    handle = torch.nn.modules.module.register_module_full_backward_hook(lambda *a: None)
    try:
        assert has_hooks(FlaggedRMSNorm(False))
    finally:
        handle.remove()


@pytest.mark.gpu
@pytest.mark.parametrize("register", ["register_full_backward_hook", "register_full_backward_pre_hook"])
def test_a_norm_with_backward_hooks_runs(register):
    """A gradient observer on a norm sees its gradient, so the module runs."""
    from test_patch_adapters import _run, build

    from forge.patching import FORWARD_MAKERS

    m, rot = build("qwen3", "attn", dtype=torch.bfloat16, device="cuda")
    seen = []
    getattr(m.k_norm, register)(lambda *a: seen.append(1))
    m.forward = FORWARD_MAKERS["lora_qkv"](m, {"fuse_qk_norm": True})
    x = torch.randn(2, 9, 512, device="cuda", dtype=torch.bfloat16)
    cos, sin = rot(x, torch.arange(9, device="cuda")[None])
    _run(m, x, ((cos, sin), None), "attn", torch.ones(2, 9, 512, device="cuda"))
    assert seen == [1]


# ---------------------------------------------------------------------------
# the rotation
# ---------------------------------------------------------------------------
def test_which_rotations_are_half_split():
    from forge.kernels.rope import forge_apply_rotary_pos_emb
    from forge.patching.kernels.lora import rotates_halves

    def of(model):
        return importlib.import_module(f"transformers.models.{model}.modeling_{model}").apply_rotary_pos_emb

    for model in ("llama", "qwen3", "qwen2", "gemma2", "gemma3", "olmo2", "t5gemma2"):
        assert rotates_halves(of(model), 128), model
    # neighbours are rotated with each other; one tensor a call; a part of the head
    for model in ("cohere", "ernie4_5", "gemma3n", "glm"):
        assert not rotates_halves(of(model), 128), model
    assert rotates_halves(forge_apply_rotary_pos_emb, 64)
    assert not rotates_halves(lambda q, k, cos, sin: (q, k), 64)


@pytest.mark.gpu
def test_fused_norms_leave_another_rotation_to_the_model(monkeypatch):
    from test_patch_adapters import MQ3, _run, build

    from forge.patching import FORWARD_MAKERS

    cohere = importlib.import_module("transformers.models.cohere.modeling_cohere")
    monkeypatch.setattr(MQ3, "apply_rotary_pos_emb", cohere.apply_rotary_pos_emb)
    m, rot = build("qwen3", "attn", dtype=torch.bfloat16, device="cuda")
    x = torch.randn(2, 9, 512, device="cuda", dtype=torch.bfloat16)
    cos, sin = rot(x, torch.arange(9, device="cuda")[None])
    outs = []
    for config in ({}, {"fuse_qk_norm": True}):
        m.forward = FORWARD_MAKERS["lora_qkv"](m, config)
        outs.append(_run(m, x, ((cos, sin), None), "attn", torch.ones(2, 9, 512, device="cuda"))[0])
    assert torch.equal(*outs)


@pytest.mark.gpu
def test_fused_projections_leave_another_rotation_to_the_model(monkeypatch):
    """A LoRA attention without norms whose model turns neighbouring columns:
    the RoPE epilogue of the fused projections is not used."""
    import copy

    from test_patch_adapters import ML, _check, _run, build

    from forge.patching import FORWARD_MAKERS

    cohere = importlib.import_module("transformers.models.cohere.modeling_cohere")
    monkeypatch.setattr(ML, "apply_rotary_pos_emb", cohere.apply_rotary_pos_emb)
    m, rot = build("llama", "attn", dtype=torch.bfloat16, device="cuda")
    m32, plain = copy.deepcopy(m).float(), copy.deepcopy(m)
    x, dy = (torch.randn(2, 9, 512, device="cuda") for _ in range(2))
    cos, sin = rot(x, torch.arange(9, device="cuda")[None])
    bf = torch.bfloat16
    r32 = _run(m32, x, ((cos.float(), sin.float()), None), "attn", dy)
    rp = _run(plain, x.to(bf), ((cos.to(bf), sin.to(bf)), None), "attn", dy)
    m.forward = FORWARD_MAKERS["lora_qkv"](m, {})
    rf = _run(m, x.to(bf), ((cos.to(bf), sin.to(bf)), None), "attn", dy)
    _check(rf[0], rp[0], r32[0], "out")
    _check(rf[1], rp[1], r32[1], "dx")


@pytest.mark.gpu
def test_fused_norms_leave_other_types_to_the_modules():
    """A float64 attention runs with the option as it does without."""
    from test_patch_adapters import _run, build

    from forge.patching import FORWARD_MAKERS

    m, rot = build("qwen3", "attn", dtype=torch.float64, device="cuda")
    x = torch.randn(2, 9, 512, device="cuda", dtype=torch.float64)
    cos, sin = rot(x, torch.arange(9, device="cuda")[None])
    outs = []
    for config in ({}, {"fuse_qk_norm": True}):
        m.forward = FORWARD_MAKERS["lora_qkv"](m, config)
        outs.append(_run(m, x, ((cos, sin), None), "attn", torch.ones(2, 9, 512, device="cuda"))[0])
    assert outs[0].dtype == torch.float64 and torch.equal(*outs)
