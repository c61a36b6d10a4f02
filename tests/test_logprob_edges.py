"""Log-probabilities and the losses built on them at the edges of what the
calls allow: sequences of no tokens, and what else `test_logprob.py` leaves out."""
import pytest
import torch

IGNORE = -100


# ---------------------------------------------------------------------------
# sequences of no tokens
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("v", [0, 1, 32000])
@pytest.mark.parametrize("n", [2, 32, 128, 1000])
def test_workspace_of_sequences_without_tokens(n, v, dtype):
    """The preference loss of empty answers still counts each answer's tokens
    (4 bytes, and two sums) and holds its log-probability (8 bytes), each array
    on 16 bytes."""
    from forge_hip import _lib as L

    assert L.forge_logp_workspace(dtype, n, 0, v) >= -(-4 * (n + 2) // 16) * 16 + 8 * n
    assert L.forge_logp_workspace(dtype, n, 0, v) <= L.forge_logp_workspace(dtype, n, 1, max(v, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("normalized", [False, True])
@pytest.mark.parametrize("pairs", [1, 64])
def test_preference_of_empty_answers(pairs, normalized, reduction):
    """Answers of no tokens have log-probability 0: h = -beta (ref_c - ref_r)."""
    from kernels.logprob import forge_preference_loss

    g = torch.Generator().manual_seed(pairs)
    ref = torch.randn(2 * pairs, generator=g)
    x = torch.zeros(2 * pairs, 0, 50, device="cuda", requires_grad=True)
    y = torch.zeros(2 * pairs, 0, device="cuda", dtype=torch.long)
    o = forge_preference_loss(x, y, ref.cuda(), beta=0.3, length_normalized=normalized, reduction=reduction)
    h = -0.3 * (ref[:pairs].double() - ref[pairs:].double())
    want = -torch.nn.functional.logsigmoid(h)
    want = {"mean": want.mean(), "sum": want.sum(), "none": want}[reduction]
    # 64-bit arithmetic and one rounding
    assert ((o.loss.detach().double().cpu() - want).abs() <= want.abs() * 2.0 ** -23).all()
    assert (o.logps == 0).all()
    rewards = -0.3 * ref.double()
    assert ((o.rewards.double().cpu() - rewards).abs() <= rewards.abs() * 2.0 ** -23).all()
    (d,) = torch.autograd.grad(o.loss, x, torch.ones_like(o.loss))
    assert d.shape == x.shape
