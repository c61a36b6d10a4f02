"""Forward-mode differentiation: the operators have no such derivatives, and a
call on a tensor with a tangent says so, as the framework's other Functions do
(a result without its tangent would be a derivative of 0)."""
import importlib

import pytest
import torch
import torch.autograd.forward_ad as fwad


def _calls(device):
    from kernels.glu_act8 import glu_act8, glu_act8_packed
    from kernels.logprob import forge_policy_loss, forge_preference_loss, forge_token_logps
    from kernels.rope import apply_qk_norm_rope

    y = torch.zeros(2, 3, dtype=torch.long, device=device)
    one = torch.ones(2, device=device)
    x = torch.randn(2, 3, 8, device=device)
    q, w = torch.randn(1, 2, 3, 8, device=device), torch.ones(8, device=device)
    c = torch.ones(1, 3, 8, device=device)
    return {
        "token_logps": (x, lambda t: forge_token_logps(t, y)),
        "preference": (x, lambda t: forge_preference_loss(t, y).loss),
        "policy": (x, lambda t: forge_policy_loss(t, y, one).loss),
        "glu gate": (x, lambda t: glu_act8(t, x)),
        "glu up": (x, lambda t: glu_act8(x, t)),
        "glu packed": (x, glu_act8_packed),
        "qk q": (q, lambda t: apply_qk_norm_rope(t, q, w, w, c, c)[0]),
        "qk k": (q, lambda t: apply_qk_norm_rope(q, t, w, w, c, c)[1]),
        "qk weight": (w, lambda t: apply_qk_norm_rope(q, q, t, w, c, c)[0]),
        "qk cos": (c, lambda t: apply_qk_norm_rope(q, q, w, w, t, c)[0]),
    }


NAMES = ["token_logps", "preference", "policy", "glu gate", "glu up", "glu packed", "qk q", "qk k", "qk weight", "qk cos"]


def _check(x, call):
    for context in (torch.no_grad(), torch.enable_grad()):
        with context, fwad.dual_level():
            call(x)  # without a tangent
            with pytest.raises(NotImplementedError, match="jvp"):
                call(fwad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused_on_the_host(name, monkeypatch):
    """The launches replaced by tensors of their results' shapes."""
    from forge_hip import _lib as L

    glu, qk, policy, preference, token_logps = (importlib.import_module(f"kernels.{m}") for m in (
        "glu_act8.glu_act8", "rope.qk_norm_rope", "logprob.policy", "logprob.preference", "logprob.token_logps"))
    monkeypatch.setattr(L, "require_gpu", lambda *a: None)
    monkeypatch.setattr(glu, "_forward", lambda g, u, act, keep: (torch.zeros(6, g.shape[-1]), torch.zeros(1)))
    monkeypatch.setattr(qk, "_forward", lambda q, k, *a: (torch.zeros(q.shape), torch.zeros(k.shape)))
    monkeypatch.setattr(token_logps, "_forward", lambda x, *a, **k: (torch.zeros(x.shape[:2]), torch.zeros(1)))
    monkeypatch.setattr(policy, "_launch", lambda x, *a: tuple(torch.zeros(s) for s in ((), x.shape[:2], x.shape[:2])))
    monkeypatch.setattr(preference.ForgePreferenceLossFunction, "forward",
                        staticmethod(lambda ctx, x, *a: tuple(torch.zeros(s) for s in ((), (2,), (2,)))))
    _check(*_calls("cpu")[name])


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name):
    _check(*_calls("cuda")[name])
