"""A patched LoRA attention that calls forge_attention (config["attention"] =
"forge"), beside the model's own implementation and an fp32 copy, and which calls
it takes."""
import copy

import pytest
import torch

pytest.importorskip("transformers")

BF16 = torch.bfloat16


def _attn(**over):
    from test_patch_adapters import build

    over = {"attn_implementation": "sdpa", **over}
    return build("llama", "attn", dtype=BF16, device=over.pop("device", "cuda"), **over)


def _patched(module, **config):
    from forge.patching import FORWARD_MAKERS

    module.forward = FORWARD_MAKERS["lora_qkv"](module, config)
    return module


def _counted(monkeypatch):
    import forge.kernels.attention as A

    calls = []
    for name in ("forge_attention", "forge_varlen_attention"):
        real = getattr(A, name)
        monkeypatch.setattr(A, name, lambda *a, _real=real, _name=name, **k: (calls.append(_name), _real(*a, **k))[1])
    return calls


def test_the_option_is_checked():
    module, _ = _attn(device="cpu")
    with pytest.raises(ValueError, match="attention must be None or 'forge'"):
        _patched(module, attention="sdpa")


def test_cpu_calls_run_the_models_implementation():
    module, rot = _attn(device="cpu")
    x = torch.randn(2, 9, 512, dtype=BF16)
    tables = rot(x, torch.arange(9)[None])
    want = _patched(copy.deepcopy(module))(x, tables, None)[0]
    assert torch.equal(_patched(module, attention="forge")(x, tables, None)[0], want)


@pytest.mark.gpu
def test_which_calls_are_taken():
    from forge.patching.kernels.lora import attention_args

    module, _ = _attn()
    q, k = (torch.zeros(2, h, 5, 128, device="cuda", dtype=BF16) for h in (4, 2))
    at = torch.tensor([0, 5], device="cuda", dtype=torch.int32)

    def args(q=q, k=k, v=None, mask=None, **kw):
        return attention_args(module, q, k, k if v is None else v, mask, kw)

    assert args() == (True, None, None)
    assert args(q=q[:, :, :1]) == (False, None, None)  # one token: every key of the cache
    assert args(position_ids=at, output_attentions=False, num_items_in_batch=3) == (True, None, None)
    # a mask, part of the queries, weights to return, an argument that is not known
    assert args(mask=torch.zeros(2, 1, 5, 5, device="cuda")) is None
    assert args(q=q[:, :, :3]) is None
    assert args(output_attentions=True) is None and args(is_causal=False, s_aux=at) is None
    # types, head sizes, devices
    assert args(q=q.float(), k=k.float()) is None and args(k=k.half()) is None and args(q=q.cpu(), k=k.cpu()) is None
    assert args(q=q[..., :4], k=k[..., :4]) is None and args(v=k[..., :64]) is None
    # sequences in a row: for the implementations that have such arguments
    assert args(q=q[:1], k=k[:1], cu_seq_lens_q=at, cu_seq_lens_k=at) is None
    module.config._attn_implementation = "flash_attention_2"
    assert args(q=q[:1], k=k[:1], cu_seq_lens_q=at, cu_seq_lens_k=at)[1] is at
    assert args(cu_seq_lens_q=at, cu_seq_lens_k=at) is None and args(q=q[:1], k=k[:1], cu_seq_lens_q=at) is None
    assert args(position_ids=at) is None and args() == (True, None, None)
    module.config._attn_implementation = "flex_attention"
    assert args() is None
    module.config._attn_implementation = "eager"  # without a mask: every key
    assert args() == (False, None, None)
    module.config._attn_implementation = "sdpa"
    module.is_causal = False
    assert args() == (False, None, None)
    module.is_causal = True
    module.sliding_window = 4
    assert args() is None
    module.sliding_window = 5
    assert args() is not None
    module.attn_logit_softcapping = 50.0
    assert args() is None
    module.attn_logit_softcapping = None
    module.attention_dropout = 0.1
    assert args() is None
    module.eval()
    assert args() is not None


@pytest.mark.gpu
@pytest.mark.parametrize("impl", ["sdpa", "eager"])
@pytest.mark.parametrize("B,S", [(2, 37), (1, 300), (3, 1)])
def test_training_beside_the_models_implementation(impl, B, S, monkeypatch):
    """Errors against an fp32 copy of at most twice the unpatched attention's, or 1% of the scale (what the
    adapters' own tests allow)."""
    from test_patch_adapters import _check, _run

    calls = _counted(monkeypatch)
    m, rot = _attn(attn_implementation=impl)
    m32, plain = copy.deepcopy(m).float(), copy.deepcopy(m)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(B, S, 512, device="cuda", generator=g) for _ in range(2))
    cos, sin = rot(x, torch.arange(S, device="cuda")[None])
    r32 = _run(m32, x, ((cos, sin), None), "attn", dy)
    rp, rf = (_run(t, x.to(BF16), ((cos.to(BF16), sin.to(BF16)), None), "attn", dy)
              for t in (_patched(plain), _patched(m, attention="forge")))
    assert calls == ["forge_attention"]
    _check(rf[0], rp[0], r32[0], "out")
    _check(rf[1], rp[1], r32[1], "dx")
    floor = _zero_gradients(m32, x, dy) if S == 1 else 0.0
    for i, (a, b, c) in enumerate(zip(rf[2], rp[2], r32[2])):
        if S == 1 and not c.any():
            assert a.abs().max() <= floor, i
        else:
            _check(a, b, c, f"lora grad {i}")


def _zero_gradients(m32, x, dy):
    """How far the gradients of the q and k factors may be from 0 where a query sees one key: p = 1 and o = v, so
    ds = sum do v - sum do o is the difference of two fp32 sums of the same 128 products in other orders, each off
    by at most 128 * 2^-24 of sum |do v|: |ds| <= 2^-16 sum |do v|.  dq = scale ds k (dk: ds q; rotations keep
    the length of pairs: sqrt 2 a value), dB = s sum over tokens dq (A x), dA = s sum (dq B) x, each with values a
    sixteenth larger at most after their bf16 roundings."""
    with torch.no_grad():
        q, k, v = (getattr(m32, n)(x) for n in ("q_proj", "k_proj", "v_proj"))
        do = (dy @ m32.o_proj.weight).view(-1, 2, 2, 128)  # [tokens, kv heads, group, D]
        ds = 2.0 ** -16 * (do * v.view(-1, 2, 1, 128)).abs().sum(-1).max()
        dq = m32.scaling * ds * 2.0 ** 0.5 * max(q.abs().max(), k.abs().max()) * 2  # (a key: of both of its heads)
        worst = 0.0
        for n in ("q_proj", "k_proj"):
            p = getattr(m32, n)
            A, B = p.lora_A["default"].weight, p.lora_B["default"].weight
            worst = max(worst, (x @ A.T).abs().max(), B.abs().sum(0).max() * x.abs().max())
        return p.scaling["default"] * x.shape[0] * dq * worst * (17 / 16) ** 4


@pytest.mark.gpu
def test_tokens_against_a_cache(monkeypatch):
    """A prompt and then single tokens with a cache: each is the same row of the whole sequence's pass, to two
    roundings of values of about 1 through a projection of 512 (some 2% of their scale)."""
    from transformers.cache_utils import DynamicCache

    calls = _counted(monkeypatch)
    m, rot = _attn()
    m = _patched(m.eval(), attention="forge")
    x = torch.randn(2, 24, 512, device="cuda", dtype=BF16)
    cos, sin = rot(x, torch.arange(24, device="cuda")[None])
    with torch.no_grad():
        whole = m(x, (cos, sin), None)[0]
        cache, parts = DynamicCache(), []
        for lo, hi in [(0, 20), (20, 21), (21, 22), (22, 23), (23, 24)]:
            parts.append(m(x[:, lo:hi], (cos[:, lo:hi], sin[:, lo:hi]), None, past_key_values=cache)[0])
    assert calls == ["forge_attention"] * 6
    got = torch.cat(parts, 1).float()
    assert (got - whole.float()).abs().max() <= 0.02 * whole.float().abs().max()


@pytest.mark.gpu
def test_sequences_packed_into_one_row(monkeypatch):
    """Every sequence of the row as it is alone: the same tiles from its first token, so the same bits of the
    attention; the projections' products differ in their last bits with the row's length."""
    calls = _counted(monkeypatch)
    m, rot = _attn()
    m.config._attn_implementation = "flash_attention_2"
    m = _patched(m.eval(), attention="forge")
    lens = [17, 1, 90]
    x = torch.randn(1, sum(lens), 512, device="cuda", dtype=BF16)
    places = torch.cat([torch.arange(n) for n in lens]).cuda()[None]
    cos, sin = rot(x, places)
    at = torch.tensor([0, 17, 18, 108], device="cuda", dtype=torch.int32)
    with torch.no_grad():
        got = m(x, (cos, sin), None, cu_seq_lens_q=at, cu_seq_lens_k=at, max_length_q=90, max_length_k=90)[0].float()
        for a, b in zip(at.tolist(), at.tolist()[1:]):
            alone = m(x[:, a:b], (cos[:, a:b], sin[:, a:b]), None)[0].float()
            assert (got[:, a:b] - alone).abs().max() <= 0.02 * alone.abs().max()
    assert calls == ["forge_varlen_attention"] + ["forge_attention"] * 3


@pytest.mark.gpu
def test_calls_that_say_whether_they_are_causal(monkeypatch):
    """is_causal of a call comes before the module's: such calls run the model's implementation, as do calls with
    any other argument that is not known, False among them."""
    from forge.patching.kernels.lora import attention_args

    calls = _counted(monkeypatch)
    module, rot = _attn()
    x = torch.randn(1, 37, 512, device="cuda", dtype=BF16)
    tables = rot(x, torch.arange(37, device="cuda")[None])
    plain, patched = _patched(copy.deepcopy(module)), _patched(copy.deepcopy(module), attention="forge")
    for value in (False, True):
        with torch.no_grad():
            want, got = (m(x, tables, None, is_causal=value)[0] for m in (plain, patched))
        assert torch.equal(got, want) and calls == []
    q, k = (torch.zeros(2, h, 5, 128, device="cuda", dtype=BF16) for h in (4, 2))
    assert attention_args(module, q, k, k, None, {"is_causal": False}) is None
    assert attention_args(module, q, k, k, None, {"some_option": False}) is None
    assert attention_args(module, q, k, k, None, {"is_causal": None, "output_attentions": False}) == (True, None, None)


@pytest.mark.gpu
def test_scales_that_forge_attention_refuses_run_the_models_implementation():
    from forge.patching.kernels.lora import attention_args

    module, _ = _attn()
    q, k = (torch.zeros(2, h, 5, 128, device="cuda", dtype=BF16) for h in (4, 2))
    for scale, taken in ((128 ** -0.5, True), (0.0, False), (-1.0, False), (1e-38, False), (1e38, False), (float("nan"), False)):
        module.scaling = scale
        assert (attention_args(module, q, k, k, None, {}) is not None) == taken, scale
