"""Token log-probabilities, preference loss and policy loss.

Tolerances, derived before the first run, with U = 2^-24, R the range of a row
of logits / temperature and V its length.  A row's fp32 sum of exponentials
has, relative to itself, the arguments' rounding ((x - max) k rounds twice: at
most 2 R U; the fp32 k is a temperature off by U: R U), 2 U of the exponential
and the additions (32 in a piece of registers, V / 8192 pieces and 20 more
across lanes, waves and pieces): a log-probability is within e = K U, K = 64 +
V / 8192 + 3 R, before it is rounded to fp32 (U of itself).  A
probability is within 2 e of itself.  Losses and coefficients are computed in
64 bits from log-probabilities that are within e, so they are within e times
their derivative; results are rounded once (finfo.eps / 2).  The hardware's
exponential gives 0 for a result below 2^-126, so a probability may be off by
that much besides.
"""
import pytest
import torch

from oracle import logprob as O

U = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
IGNORE = -100


def _logits(n, s, v, dtype, seed=0, std=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, s, v, generator=g) * std
    y = torch.randint(0, v, (n, s), generator=g)
    x.scatter_add_(-1, y.unsqueeze(-1), torch.randn(n, s, 1, generator=g) + 3.0)
    return x.to(dtype), y


def _mask(y, seed=1, keep=0.7):
    g = torch.Generator().manual_seed(seed)
    return torch.where(torch.rand(y.shape, generator=g) < keep, y, IGNORE)


def _e(x, temperature=1.0):
    """The bound e of each row's log-probability."""
    z = x.double() / temperature
    return (64 + x.shape[-1] / 8192 + 3 * (z.amax(-1) - z.amin(-1))) * U


def _near(got, ref, bound, what):
    got = got.double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = ((got - ref).abs() - bound).max().item() if got.numel() else -1
    assert off <= 0, f"{what}: off by {off:.3e} more than the bound"


def _near_logps(got, x, y, temperature=1.0):
    ref = O.token_logps(x, y, temperature=temperature)
    _near(got, ref, torch.where(y == IGNORE, 0.0, _e(x, temperature) + ref.abs() * U), "logps")
    return ref


def _near_dlogits(got, x, y, coef, coef_off, temperature=1.0):
    """coef within coef_off (both [N, S])."""
    ref = O.dlogits(x, y, coef, temperature=temperature)
    e = _e(x, temperature).unsqueeze(-1)
    c, off = coef.abs().unsqueeze(-1) / temperature, (coef_off / temperature).unsqueeze(-1)
    p = (x.double() / temperature).softmax(-1)
    hot = torch.zeros_like(p).scatter_(-1, y.clamp(min=0).unsqueeze(-1), 1.0)
    size = torch.where(hot == 1, 1 - p, p)
    bound = c * 2 * e * torch.where(hot == 1, torch.ones_like(p), p) + off * size + 8 * U * ref.abs() + c * 2.0 ** -126
    eps = torch.finfo(got.dtype).eps
    bound = bound * (1 + eps) + ref.abs() * eps / 2 + torch.finfo(got.dtype).smallest_normal * eps
    _near(got, ref, torch.where((y == IGNORE).unsqueeze(-1), 0.0, bound), "dlogits")


# ---------------------------------------------------------------------------
# the oracle and the refusals (CPU)
# ---------------------------------------------------------------------------
def test_oracle_token_gradient_against_differences():
    x, y = _logits(2, 3, 7, torch.float64)
    y = _mask(y, keep=0.6)
    x.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda t: O.token_logps(t, y, temperature=0.7), x)
    g = torch.Generator().manual_seed(3)
    c = torch.randn(2, 3, generator=g, dtype=torch.float64)
    (d,) = torch.autograd.grad(O.token_logps(x, y, temperature=0.7), x, c)
    torch.testing.assert_close(O.dlogits(x.detach(), y, c, temperature=0.7), d, rtol=1e-10, atol=1e-12)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("kind,smoothing,normalized", [("sigmoid", 0.0, False), ("sigmoid", 0.1, True),
                                                       ("hinge", 0.0, False), ("ipo", 0.0, True)])
def test_oracle_preference_against_differences(kind, smoothing, normalized, reduction):
    g = torch.Generator().manual_seed(0)
    lp = torch.randn(6, 5, generator=g, dtype=torch.float64).requires_grad_(True)
    kept = torch.rand(6, 5, generator=g) < 0.7
    kept[2] = False
    ref = torch.randn(6, generator=g)
    up = torch.randn(3, generator=g, dtype=torch.float64)

    def loss(t):
        out = O.preference(t, kept, ref, 0.3, smoothing, kind, normalized, reduction)[0]
        return (out * up).sum() if reduction == "none" else out

    assert torch.autograd.gradcheck(loss, lp)
    (d,) = torch.autograd.grad(loss(lp), lp)
    coef = O.preference(lp.detach(), kept, ref, 0.3, smoothing, kind, normalized, reduction)[3]
    if reduction == "none":
        coef = coef * torch.cat([up, up]).unsqueeze(-1)
    torch.testing.assert_close(coef, d, rtol=1e-9, atol=1e-12)


@pytest.mark.parametrize("reduction", ["mean", "sum", "sequence"])
@pytest.mark.parametrize("old,ref", [(False, False), (True, False), (False, True), (True, True)])
def test_oracle_policy_against_differences(old, ref, reduction):
    g = torch.Generator().manual_seed(1)
    lp = torch.randn(4, 6, generator=g, dtype=torch.float64).requires_grad_(True)
    kept = torch.rand(4, 6, generator=g) < 0.7
    kept[1] = False
    adv = torch.randn(4, 1, generator=g).expand(4, 6)
    o = lp.detach() + 0.3 * torch.randn(4, 6, generator=g, dtype=torch.float64) if old else None
    r = lp.detach() + 0.3 * torch.randn(4, 6, generator=g, dtype=torch.float64) if ref else None

    here = lp.detach().clone()

    def loss(t):
        # without old log-probabilities the ratio is 1 in value and the log-probability's in slope
        return O.policy(t, kept, adv, here if o is None else o, r, 0.2, 0.28, 0.05, reduction)[0]

    assert torch.autograd.gradcheck(loss, lp)
    (d,) = torch.autograd.grad(loss(lp), lp)
    value, _, coef = O.policy(lp.detach(), kept, adv, o, r, 0.2, 0.28, 0.05, reduction)
    torch.testing.assert_close(value, loss(lp).detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(coef, d, rtol=1e-9, atol=1e-12)


def test_refusals():
    from kernels.logprob import forge_policy_loss, forge_preference_loss, forge_token_logps

    x, y = torch.zeros(4, 3, 8), torch.zeros(4, 3, dtype=torch.long)
    adv = torch.zeros(4)
    for call in (forge_token_logps, forge_preference_loss, lambda a, b, **k: forge_policy_loss(a, b, adv, **k)):
        with pytest.raises(ValueError, match="one target a row"):
            call(x, y[:, :2])
        with pytest.raises(TypeError, match="fp16, bf16 or fp32"):
            call(x.double(), y)
        with pytest.raises(TypeError, match="integer tensor"):
            call(x, y.float())
        with pytest.raises(ValueError, match="no columns"):
            call(x[..., :0], y)
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call(x, y)
    for t in (0.0, -1.0, float("inf"), float("nan"), 1e-7):
        with pytest.raises(ValueError, match="temperature"):
            forge_token_logps(x, y, temperature=t)

    def pref(error, match, *a, **k):
        with pytest.raises(error, match=match):
            forge_preference_loss(*(a or (x, y)), **k)

    pref(ValueError, r"2 \* pairs", x[:3], y[:3])
    pref(ValueError, r"2 \* pairs", x[0], y[0])
    pref(ValueError, "loss_type", loss_type="dpo")
    pref(ValueError, "reduction", reduction="sequence")
    pref(ValueError, "beta", beta=0.0)
    pref(ValueError, "label_smoothing must", label_smoothing=1.5)
    pref(ValueError, "belongs to", label_smoothing=0.1, loss_type="ipo")
    pref(ValueError, "ref_logps must have shape", ref_logps=torch.zeros(2))
    pref(TypeError, "ref_logps must be floating", ref_logps=torch.zeros(4, dtype=torch.long))
    pref(ValueError, "inplace", torch.zeros(4, 1, 8).expand(4, 3, 8), y, inplace=True)

    def policy(error, match, logits=x, target=y, a=adv, **k):
        with pytest.raises(error, match=match):
            forge_policy_loss(logits, target, a, **k)

    policy(ValueError, r"\[sequences, seq, vocab\]", x[0], y[0])
    policy(ValueError, "advantages must have shape", a=adv[:2])
    policy(ValueError, "advantages must have shape", a=torch.zeros(4, 2))
    policy(ValueError, "old_logps must have shape", old_logps=adv)
    policy(ValueError, "reduction", reduction="none")
    policy(ValueError, "clip_low", clip_low=1.5)
    policy(ValueError, "clip_low", clip_high=-0.1)
    policy(ValueError, "needs ref_logps", kl_coef=0.1)
    policy(ValueError, "not a leaf", torch.zeros(4, 3, 8, requires_grad=True), inplace=True)
    policy(ValueError, "inplace", torch.zeros(4, 8, 3).transpose(1, 2), inplace=True)
    policy(ValueError, "inplace", torch.zeros(4, 30).as_strided((4, 3, 8), (30, 4, 1)), inplace=True)


def test_target_checks():
    from kernels.logprob._rows import check_inplace, check_targets

    check_targets(torch.tensor([0, 7, IGNORE]), IGNORE, 8)
    check_targets(torch.tensor([], dtype=torch.long), IGNORE, 8)
    check_targets(torch.tensor([1000, 3]), 1000, 8)
    for bad in ([8], [-1], [IGNORE, -2]):
        with pytest.raises(IndexError):
            check_targets(torch.tensor(bad), IGNORE, 8)
    x = torch.zeros(4, 6, 8)
    for ok in (x, x[:, 1:3], x[::2], x.transpose(0, 1), x[..., :5], x[:1, :1], x[:, :1].expand(4, 1, 8)):
        check_inplace(ok)


def test_c_entry_errors():
    from forge_hip import _lib as L

    def rows(n=2, s=3, v=8, dtype=2):
        return (dtype, 16, 24, 8, n, s, v, 16, 3, 1, IGNORE)

    assert L.forge_logp_workspace(2, 2, 3, 8) > 0
    assert L.forge_token_logps_fwd(*rows(dtype=3), 1.0, 16, None, 16, None) == 2
    assert L.forge_token_logps_fwd(*rows(), 0.0, 16, None, 16, None) == 1 and b"temperature" in L.forge_last_error()
    assert L.forge_token_logps_fwd(*rows(n=-1), 1.0, 16, None, 16, None) == 1
    assert L.forge_token_logps_fwd(*rows(v=0), 1.0, 16, None, 16, None) == 1 and b"columns" in L.forge_last_error()
    assert L.forge_token_logps_fwd(*rows(n=1 << 20, s=1 << 20), 1.0, 16, None, 16, None) == 2
    assert L.forge_token_logps_fwd(*rows(n=0), 1.0, 16, None, 16, None) == 0
    assert L.forge_token_logps_bwd(*rows(), 1.0, 16, 16, 16, 3, 1, 16, 0, 0, 16, 24, 8, None) == 1
    assert b"up_count" in L.forge_last_error()
    pref = (None, 0.1, 0.0, 0, 0, 1, 16, 16, 16, 16, 16, 16, 16, None)
    assert L.forge_preference_fwd(*rows(n=0), *pref) == 1 and b"no pairs" in L.forge_last_error()
    assert L.forge_preference_fwd(*rows(), None, 0.1, 0.0, 3, 0, 1, *pref[6:]) == 1 and b"kind" in L.forge_last_error()
    assert L.forge_preference_fwd(*rows(), None, 0.1, 0.0, 0, 0, 3, *pref[6:]) == 1
    assert L.forge_token_logps_fwd(*rows(), 1.0, None, None, 16, None) == 1 and b"NULL" in L.forge_last_error()
    assert L.forge_token_logps_bwd(*rows(), 1.0, 16, None, 16, 3, 1, None, 0, 1, 16, 24, 8, None) == 1
    assert L.forge_preference_fwd(*rows(), *pref[:-2], None, None) == 1 and b"NULL" in L.forge_last_error()
    none = (None, 0, 0)
    rc = L.forge_policy_loss(*rows(), 1.0, None, 1, 0, *none, *none, 0.2, 0.2, 0.0, 1, 16, 16, 16, None, 0, 0, 16, None)
    assert rc == 1 and b"NULL" in L.forge_last_error()
    rc = L.forge_policy_loss(*rows(), 1.0, 16, 1, 0, *none, *none, 0.2, 0.2, 0.0, 0, 16, 16, 16, None, 0, 0, 16, None)
    assert rc == 1 and b"reduction" in L.forge_last_error()


# ---------------------------------------------------------------------------
# token log-probabilities
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("n,s,v", [(1, 1, 1), (1, 1, 3), (2, 3, 7), (1, 5, 8), (3, 4, 33), (2, 2, 1000), (5, 3, 2049),
                                   (1, 2, 9001), (2, 3, 50257), (1, 3, 128256)])
def test_token_logps(n, s, v, dtype):
    from kernels.logprob import forge_token_logps

    x, y = _logits(n, s, v, dtype, seed=v)
    if n * s > 3:
        y = _mask(y)
    temperature = 1.0 if v % 2 else 0.7
    xg = x.cuda().requires_grad_(True)
    got = forge_token_logps(xg, y.cuda(), temperature=temperature)
    assert got.dtype == FP32
    _near_logps(got.detach(), x, y, temperature)
    g = torch.Generator().manual_seed(2)
    c = torch.randn(n, s, generator=g)
    (d,) = torch.autograd.grad(got, xg, c.cuda())
    assert d.dtype == dtype
    _near_dlogits(d, x, y, c.double(), torch.zeros(n, s), temperature)
    with torch.no_grad():
        assert torch.equal(forge_token_logps(xg, y.cuda(), temperature=temperature), got)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,v", [(1, 30011), (9, 30011), (1100, 30011), (3000, 30011), (700, 1003), (513, 8195)])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
def test_token_logps_row_counts(rows, v, dtype):
    """From rows that are split over many workgroups to rows of their own, long
    ones and short ones."""
    from kernels.logprob import forge_token_logps

    x, y = _logits(rows, 1, v, dtype, seed=rows)
    xg = x.cuda().requires_grad_(True)
    got = forge_token_logps(xg, y.cuda())
    _near_logps(got.detach(), x, y)
    (d,) = torch.autograd.grad(got, xg, torch.ones(rows, 1, device="cuda"))
    last = slice(max(0, rows - 5), rows)
    _near_dlogits(d[last], x[last], y[last], torch.ones_like(y[last]).double(), torch.zeros(y[last].shape))
    # rows of (onehot - p) add up to 0 but for each term's rounding
    assert d.double().sum(-1).abs().max() <= 2 * torch.finfo(dtype).eps + 2 * _e(x).max()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(11,), (5, 11), (2, 3, 4, 11)])
def test_leading_shapes(shape):
    from kernels.logprob import forge_token_logps

    g = torch.Generator().manual_seed(0)
    x = torch.randn(shape, generator=g)
    y = torch.randint(0, 11, shape[:-1], generator=g)
    got = forge_token_logps(x.cuda(), y.cuda().int())
    assert got.shape == y.shape
    torch.testing.assert_close(got.cpu(), x.log_softmax(-1).gather(-1, y.unsqueeze(-1)).squeeze(-1), rtol=0,
                               atol=float(_e(x).max()) + 8 * U)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
def test_strided_logits_and_targets(dtype):
    """Shifted slices, columns of a padded vocabulary (rows off 16 bytes),
    sequence-first memory, a transposed vocabulary, expanded gradients."""
    from kernels.logprob import forge_token_logps

    big, y = _logits(3, 6, 517, dtype)
    yg = y.cuda()
    views = [lambda t: t[:, :-1], lambda t: t[..., :509], lambda t: t[..., 3:510], lambda t: t[::2],
             lambda t: t.transpose(0, 1), lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)]
    for view in views:
        x = view(big)
        t = (y.transpose(0, 1) if x.shape[0] == 6 else y[:x.shape[0], :x.shape[1]] if x.shape[0] == 3 else y[::2])
        t = t.clamp(max=x.shape[-1] - 1)
        tg = yg.new_empty(t.shape[1], t.shape[0]).T.copy_(t)  # sequence-first targets too
        xg = view(big.cuda().requires_grad_(True))
        got = forge_token_logps(xg, tg)
        _near_logps(got.detach(), x, t)
        (d,) = torch.autograd.grad(got.sum(), xg)
        _near_dlogits(d, x, t, torch.ones(t.shape, dtype=torch.float64), torch.zeros(t.shape))


@pytest.mark.gpu
def test_masked_and_infinite_logits():
    """-inf columns, rows of nothing else, +inf, NaN, a target at -inf; and
    nothing of an ignored row counts."""
    from kernels.logprob import forge_token_logps

    x, y = _logits(1, 8, 300, FP32)
    inf = float("inf")
    x[0, 0, 10:250] = -inf
    x[0, 1] = -inf
    x[0, 2, 5] = inf
    x[0, 3, 7] = float("nan")
    y[0, 0] = 255
    y[0, 4], x[0, 4, 3] = 3, -inf
    x[0, 5] = float("nan")
    y[0, 5] = IGNORE
    x[0, 6] = -1e30
    xg = x.cuda().requires_grad_(True)
    got = forge_token_logps(xg, y.cuda())
    ref = x.double().log_softmax(-1).gather(-1, y.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    assert got[0, [1, 2, 3]].isnan().all() and ref[0, [1, 2, 3]].isnan().all()
    assert got[0, 4] == -inf and got[0, 5] == 0
    keep = [0, 6, 7]
    assert ((got[0, keep].cpu().double() - ref[0, keep]).abs() <= 200 * U + ref[0, keep].abs() * U).all()
    (d,) = torch.autograd.grad(got, xg, torch.ones_like(got))
    assert (d[0, 0, 10:250] == 0).all() and not d[0, [0, 4, 5, 6, 7]].isnan().any() and (d[0, 5] == 0).all()
    assert d[0, 1:4].isnan().any(-1).all()
    # an incoming gradient of 0 gives a row of zeros whatever the row holds
    got = forge_token_logps(xg, y.cuda())
    (d,) = torch.autograd.grad(got, xg, torch.zeros_like(got))
    assert (d == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1e-6, 0.01, 100.0, 1e6])
@pytest.mark.parametrize("rows", [3, 600])
def test_extreme_temperatures(temperature, rows):
    """From all of the probability on the largest logit to the same on each."""
    from kernels.logprob import forge_policy_loss, forge_token_logps

    x, y = _logits(1, rows, 515, BF16)
    xg, yg = x.cuda().requires_grad_(True), y.cuda()
    got = forge_token_logps(xg, yg, temperature=temperature)
    ref = O.token_logps(x, y, temperature=temperature)
    # the exponents' rounding is relative to the scaled differences, which are as large as the result here
    bound = _e(x, temperature) + ref.abs() * 2 * U
    _near(got.detach(), ref, bound, "logps")
    o = forge_policy_loss(xg, yg, torch.ones(1, device="cuda"), temperature=temperature)
    _near(o.logps, ref, bound, "policy logps")
    (d,) = torch.autograd.grad(o.loss, xg)
    if temperature >= 0.01:
        w = -1.0 / rows
        _near_dlogits(d, x, y, torch.full((1, rows), w).double(), torch.full((1, rows), 2 * U * abs(w)), temperature)
    else:
        assert not d.isnan().any()


@pytest.mark.gpu
def test_targets_out_of_range():
    from kernels.logprob import forge_policy_loss, forge_preference_loss, forge_token_logps

    x, y = _logits(2, 4, 50, BF16)
    bad = y.clone()
    bad[0, 1], bad[1, 2] = 50, -3
    xg = x.cuda().requires_grad_(True)
    got, good = forge_token_logps(xg, bad.cuda()), forge_token_logps(xg, y.cuda())
    (d,) = torch.autograd.grad(got.nansum(), xg, retain_graph=True)
    (d1,) = torch.autograd.grad(got, xg, torch.ones_like(got))
    wrong = torch.zeros(2, 4, dtype=torch.bool)
    wrong[0, 1] = wrong[1, 2] = True
    assert got[wrong].isnan().all() and torch.equal(got[~wrong], good[~wrong])
    assert d1[wrong].isnan().all() and not d1[~wrong].isnan().any() and not d[~wrong].isnan().any()
    for call in (lambda **k: forge_token_logps(xg, bad.cuda(), **k),
                 lambda **k: forge_preference_loss(xg, bad.cuda(), **k).loss,
                 lambda **k: forge_policy_loss(xg, bad.cuda(), torch.ones(2, device="cuda"), **k).loss):
        assert call().isnan().any()
        with pytest.raises(IndexError, match="targets must be"):
            call(validate_targets=True)


# ---------------------------------------------------------------------------
# preference loss
# ---------------------------------------------------------------------------
def _preference_case(x, y, ref, beta, smoothing, kind, normalized, reduction, inplace=False, scale=None):
    from kernels.logprob import forge_preference_loss

    leaf = x.cuda().requires_grad_(True)
    xg = leaf * 1.0  # logits are a layer's output
    o = forge_preference_loss(xg, y.cuda(), None if ref is None else ref.cuda(), beta=beta, label_smoothing=smoothing,
                              loss_type=kind, length_normalized=normalized, reduction=reduction, inplace=inplace)
    assert o.loss.requires_grad and not o.logps.requires_grad and not o.rewards.requires_grad
    up = torch.ones_like(o.loss) if scale is None else scale.cuda()
    (d,) = torch.autograd.grad(o.loss, leaf, up)
    kept = y != IGNORE
    lp = O.token_logps(x, y)
    loss, seq, rewards, coef = O.preference(lp, kept, ref, beta, smoothing, kind, normalized, reduction)
    pairs = len(seq) // 2
    n = kept.sum(-1).double().clamp(min=1) if normalized else torch.ones(2 * pairs).double()
    e = torch.where(kept, _e(x) + 0 * lp, 0.0).sum(-1) / n   # of a sequence's log-probability
    _near(o.logps, seq, e + seq.abs() * U, "seq_logps")
    _near(o.rewards, rewards, beta * e + rewards.abs() * U, "rewards")
    e_h = e[:pairs] + e[pairs:]                               # of chosen less rejected
    over = rewards / beta
    t = over[:pairs] - over[pairs:] - 0.5 / beta
    first = {"sigmoid": beta * torch.ones_like(t), "hinge": beta * torch.ones_like(t), "ipo": 2 * t.abs() + e_h}[kind]
    second = {"sigmoid": beta * beta / 4, "hinge": 0.0, "ipo": 2.0}[kind]
    w = 1.0 / pairs if reduction == "mean" else 1.0
    off = first * e_h * w
    _near(o.loss.detach(), loss, (off if reduction == "none" else off.sum()) + loss.abs() * U, "loss")
    coef_off = (torch.cat([e_h, e_h]) * second * w / n).unsqueeze(-1) + 2 * U * coef.abs()
    upc = up.double().cpu()
    upc = torch.cat([upc, upc]).unsqueeze(-1) if reduction == "none" else upc
    _near_dlogits(d, x, y, coef * upc, coef_off * upc.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("kind,smoothing,normalized,reduction", [
    ("sigmoid", 0.0, False, "mean"), ("sigmoid", 0.2, True, "sum"), ("sigmoid", 0.1, False, "none"),
    ("hinge", 0.0, True, "mean"), ("ipo", 0.0, True, "mean"), ("ipo", 0.0, False, "none")])
@pytest.mark.parametrize("pairs,s,v", [(1, 1, 5), (3, 7, 101), (2, 40, 5001), (5, 3, 32000)])
def test_preference(pairs, s, v, kind, smoothing, normalized, reduction, dtype):
    x, y = _logits(2 * pairs, s, v, dtype, seed=s)
    y = _mask(y) if s > 1 else y
    if pairs == 5:
        y[3] = IGNORE  # an answer of no tokens
    g = torch.Generator().manual_seed(4)
    lp = O.token_logps(x, y).sum(-1)
    if normalized:
        lp = lp / (y != IGNORE).sum(-1).clamp(min=1)
    ref = (lp + torch.randn(2 * pairs, generator=g)).float()
    scale = torch.randn(pairs, generator=g) if reduction == "none" else torch.tensor(0.37)
    _preference_case(x, y, ref, 0.3, smoothing, kind, normalized, reduction, scale=scale)


@pytest.mark.gpu
def test_preference_long_answers_without_reference():
    """Sums of 3000 log-probabilities a sequence, 6 pairs, no reference; far
    margins saturate without overflow."""
    x, y = _logits(12, 3001, 70, FP32, seed=8)
    _preference_case(x, y, None, 0.1, 0.0, "sigmoid", False, "mean")
    _preference_case(x, _mask(y), None, 50.0, 0.0, "sigmoid", False, "sum")


@pytest.mark.gpu
def test_preference_extreme_margins():
    """A margin whose exponential leaves fp32 and fp64: the loss is the margin
    or 0, never infinite."""
    from kernels.logprob import forge_preference_loss

    x, y = _logits(2, 3, 40, FP32)
    for sign in (1.0, -1.0):
        ref = torch.tensor([1e5 * sign, -1e5 * sign]).cuda()
        xg = x.cuda().requires_grad_(True)
        o = forge_preference_loss(xg, y.cuda(), ref, beta=1.0)
        (d,) = torch.autograd.grad(o.loss, xg)
        assert d.isfinite().all()
        if sign > 0:
            torch.testing.assert_close(o.loss.item(), 2e5, rtol=1e-3, atol=0)
        else:
            assert o.loss.item() == 0.0 and (d == 0).all()


@pytest.mark.gpu
def test_preference_inplace():
    from kernels.logprob import forge_preference_loss

    x, y = _logits(4, 9, 777, BF16)
    y = _mask(y).cuda()
    ref = torch.zeros(4).cuda()
    a, b = x.cuda().requires_grad_(True), x.cuda().requires_grad_(True)
    la, lb = a * 1.0, b * 1.0
    oa, ob = forge_preference_loss(la, y, ref), forge_preference_loss(lb, y, ref, inplace=True)
    assert torch.equal(oa.loss, ob.loss) and torch.equal(la, lb)
    (da,) = torch.autograd.grad(oa.loss, a, retain_graph=True)
    (again,) = torch.autograd.grad(oa.loss, a)
    (dlb,) = torch.autograd.grad(ob.loss, lb, retain_graph=True)
    assert torch.equal(da, again) and torch.equal(da, dlb) and dlb.data_ptr() == lb.data_ptr()
    with pytest.raises(RuntimeError, match="runs once"):
        torch.autograd.grad(ob.loss, lb)
    # what else saved the logits is told that they are gone; logits changed since the forward are refused
    lc = x.cuda().requires_grad_(True) * 1.0
    square = (lc * lc).sum()
    forge_preference_loss(lc, y, ref, inplace=True).loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        square.backward()
    for inplace in (False, True):
        ld = x.cuda().requires_grad_(True) * 1.0
        o = forge_preference_loss(ld, y, ref, inplace=inplace)
        ld.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified"):
            o.loss.backward()


# ---------------------------------------------------------------------------
# policy loss
# ---------------------------------------------------------------------------
def _policy_inputs(x, y, temperature, seed, per_token=False):
    g = torch.Generator().manual_seed(seed)
    lp = O.token_logps(x, y, temperature=temperature)
    n, s = y.shape
    adv = torch.randn(n, s, generator=g) if per_token else torch.randn(n, generator=g)
    old = (lp + 0.3 * torch.randn(n, s, generator=g)).float()
    ref = (lp + 0.5 * torch.randn(n, s, generator=g)).float()
    return adv, old, ref


def _policy_case(x, y, adv, old, ref, beta, temperature, reduction, inplace=False, scale=1.0, view=lambda t: t):
    from kernels.logprob import forge_policy_loss

    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    leaf = x.cuda().requires_grad_(True)
    xg = view(leaf * 1.0)
    before = xg.detach().clone()
    o = forge_policy_loss(xg, y.cuda(), cuda(adv), cuda(old), cuda(ref), clip_low=0.2, clip_high=0.28, kl_coef=beta,
                          temperature=temperature, reduction=reduction, inplace=inplace)
    if not inplace:
        assert torch.equal(before, xg)
    with torch.no_grad():
        plain = forge_policy_loss(before, y.cuda(), cuda(adv), cuda(old), cuda(ref), clip_low=0.2, clip_high=0.28,
                                  kl_coef=beta, temperature=temperature, reduction=reduction)
    if y.numel() < 256:  # (a large call with a gradient holds its rows on chip: other roundings)
        assert torch.equal(plain.loss, o.loss) and torch.equal(plain.logps, o.logps) and torch.equal(plain.kl, o.kl)
    else:
        _near_logps(plain.logps, view(x), y, temperature)
    (d,) = torch.autograd.grad(o.loss, leaf, torch.tensor(scale, device="cuda"))
    x, d = view(x), view(d)
    kept = y != IGNORE
    lp = _near_logps(o.logps, x, y, temperature)
    a2 = adv.unsqueeze(1).expand(y.shape) if adv.dim() == 1 else adv
    loss, kl, coef = O.policy(lp, kept, a2, old, ref, 0.2, 0.28, beta, reduction)
    e = torch.where(kept, _e(x, temperature), 0.0)
    # |dloss/dlogp| and its change with logp, before the weights
    ratio = torch.ones_like(lp) if old is None else (lp - old.double()).exp()
    far = torch.zeros_like(lp) if ref is None else (ref.double() - lp)
    slope = (a2.double() * ratio).abs() + beta * torch.expm1(far).abs()
    bend = (a2.double() * ratio).abs() * (0 if old is None else 1) + beta * far.exp()
    _, _, w = O.policy(lp, kept, -torch.ones_like(a2), lp, None, 0.2, 0.28, 0.0, reduction)  # coefficient w of A = -1
    _near(o.loss.detach(), loss, (w * (slope + bend * e) * e).sum() * 1.01 + (w * slope).sum() * U + loss.abs() * U, "loss")
    if ref is not None:
        _near(o.kl, kl, (torch.expm1(far).abs() + far.exp() * e) * e * 1.01 + kl * 2 * U, "kl")
    off = w * bend * e * 1.01 + 2 * U * coef.abs()
    if scale != 1.0:  # a second rounding of the stored gradient
        eps = torch.finfo(d.dtype).eps
        d1 = O.dlogits(x, y, coef, temperature=temperature) * scale
        bound = d1.abs() * eps * 1.1 + abs(scale) * (3 * e + 12 * U).unsqueeze(-1) * coef.abs().unsqueeze(-1) / temperature
        bound = bound + abs(scale) * off.unsqueeze(-1) / temperature + torch.finfo(d.dtype).smallest_normal
        return _near(d, d1, bound, "scaled dlogits")
    _near_dlogits(d, x, y, coef, off, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("reduction", ["mean", "sequence", "sum"])
@pytest.mark.parametrize("old,ref,beta,per_token", [(True, True, 0.04, False), (False, True, 0.5, True),
                                                    (True, False, 0.0, True), (False, False, 0.0, False),
                                                    (True, True, 0.0, False)])
@pytest.mark.parametrize("n,s,v", [(1, 1, 9), (4, 13, 260), (3, 5, 32000), (40, 3, 65), (1, 700, 40)])
def test_policy(n, s, v, old, ref, beta, per_token, reduction, dtype):
    x, y = _logits(n, s, v, dtype, seed=n)
    if n > 1:
        y = _mask(y)
        y[1] = IGNORE  # a sequence of no tokens
    temperature = 0.8 if n == 4 else 1.0
    adv, o, r = _policy_inputs(x, y, temperature, seed=s, per_token=per_token)
    _policy_case(x, y, adv, o if old else None, r if ref else None, beta, temperature, reduction)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,v", [(BF16, 1000), (BF16, 32000), (BF16, 50257), (FP16, 65544), (BF16, 128256),
                                     (BF16, 131072), (BF16, 131080), (FP32, 32000), (FP16, 8), (BF16, 4104), (BF16, 8199),
                                     (FP16, 8192), (BF16, 4095), (FP32, 4100), (FP32, 1001)])
def test_policy_many_rows(dtype, v):
    """Enough rows that every row has a workgroup of its own."""
    n, s = 6, 350
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.empty(n, s, v, device="cuda", dtype=dtype).normal_(0, 2, generator=g)
    y = torch.randint(0, v, (n, s), device="cuda", generator=g)
    y[:, :17] = IGNORE
    y[2] = IGNORE
    from kernels.logprob import forge_policy_loss, forge_token_logps

    adv = torch.randn(n, device="cuda", generator=g)
    base = forge_token_logps(x, y)
    old = base + 0.2 * torch.randn(n, s, device="cuda", generator=g)
    ref = base + 0.2 * torch.randn(n, s, device="cuda", generator=g)
    xg = x.requires_grad_(True)
    o = forge_policy_loss(xg, y, adv, old, ref, kl_coef=0.1)
    (d,) = torch.autograd.grad(o.loss, xg)
    pick = torch.tensor([[0, 0], [0, 17], [1, 200], [2, 30], [3, 349], [5, 349], [5, 348]])
    xs, ys = x.detach()[pick[:, 0], pick[:, 1]].cpu().unsqueeze(0), y[pick[:, 0], pick[:, 1]].cpu().unsqueeze(0)
    take = lambda t: t[pick[:, 0], pick[:, 1]].unsqueeze(0)  # noqa: E731
    lp = _near_logps(take(o.logps).cpu(), xs, ys)
    kept = (y != IGNORE).cpu()
    loss, _, coef = O.policy(o.logps.double().cpu(), kept, adv.cpu().unsqueeze(1).expand(n, s), old.cpu(), ref.cpu(), 0.2,
                             0.2, 0.1, "mean")
    # the oracle's losses from the fp32 log-probabilities: U of each and e of what precedes them
    e = (64 + v / 8192 + 40) * U + base.abs().max().item() * U
    slope = (adv.abs().max().item() * 3 + 0.3)
    _near(o.loss.detach(), loss, slope * e + loss.abs() * U, "loss")
    tokens = kept.sum().item()
    _near_dlogits(take(d), xs, ys, take(coef), torch.full(ys.shape, slope * e / tokens))
    assert lp.shape == ys.shape and (d[y == IGNORE] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=str)
@pytest.mark.parametrize("v,inplace", [(5, False), (3003, True), (8001, False), (20000, False), (40001, True), (70000, True),
                                       (120000, False)])
def test_policy_awkward_rows(v, inplace, dtype):
    """Rows of negative values, of a mask's lowest values, with infinities and
    NaN, targets out of range and clipped tokens, in a batch large enough for a
    row to a workgroup: a call of its own for each must give the same."""
    from kernels.logprob import forge_policy_loss

    s, inf, low = 600, float("inf"), torch.finfo(dtype).min
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.empty(1, s, v, device="cuda", dtype=dtype).normal_(0, 2, generator=g)
    y = torch.randint(0, v, (1, s), device="cuda", generator=g)
    x[0, 0] = -x[0, 0].abs() - 3          # nothing but negative values
    x[0, 1] = low                          # nothing but the lowest value
    x[0, 2] = low
    x[0, 2, v // 2] = 1.5                  # one value left, and it is not the target's
    x[0, 3] = -inf
    x[0, 4, 1] = inf
    x[0, 5, v - 1] = float("nan")
    x[0, 6, v // 3:] = -inf
    y[0, 6] = 0
    x[0, 7, y[0, 7]] = -inf                # the target is masked
    x[0, 8], x[0, 8, y[0, 8]] = low / 2, low / 4
    y[0, 9], y[0, 10] = v, -7
    x[0, 11] = 0.0
    x[0, 12] = torch.finfo(dtype).max
    y[0, 13], y[0, 14] = v - 1, 0
    y[0, 15:40] = IGNORE
    adv = torch.empty(1, s, device="cuda").normal_(generator=g)
    old = torch.full((1, s), -11.0, device="cuda")
    old[0, 41], adv[0, 41] = -200.0, 1.0   # the ratio is past its clip: no gradient
    ref = torch.full((1, s), -10.0, device="cuda")
    ref[0, 41] = 0.0

    def call(rows, inplace):
        leaf = x[:, rows].clone().requires_grad_(True)
        t = leaf * 1.0
        o = forge_policy_loss(t, y[:, rows], adv[:, rows], old[:, rows], reduction="sum", inplace=inplace)
        return (o, *torch.autograd.grad(o.loss, leaf))

    o, d = call(slice(None), inplace)
    assert o.loss.isnan() and (d[0, 15:40] == 0).all() and (d[0, 41] == 0).all()
    rows = list(range(15)) + [41, 42, 599]
    for r in rows:
        one, d1 = call(slice(r, r + 1), False)
        a, b = o.logps[0, r], one.logps[0, 0]
        assert a == b or (a.isnan() and b.isnan()) or abs(a - b) <= 4 * float(_e(torch.tensor([[0.0, 20.0]])).max()) + \
            abs(b) * 2 * U, (r, a, b)
        assert torch.equal(d[0, r].isnan(), d1[0, 0].isnan()), r
        eps = torch.finfo(dtype).eps
        off = (d[0, r].float() - d1[0, 0].float()).abs() - d1[0, 0].float().abs() * eps * 1.1
        # both within e of a row's log-probability, times the coefficient A r
        e = float(_e(x[0, r].float().cpu().unsqueeze(0)))
        if b.isfinite() and e < 1.0:
            off = off - 4 * e * (adv[0, r].abs() * (b - old[0, r]).exp())
        fin = d1[0, 0].isfinite()
        assert (off[fin] <= torch.finfo(dtype).smallest_normal).all(), (r, off[fin].max())
        assert torch.equal(d[0, r][~fin & ~d1[0, 0].isnan()], d1[0, 0][~fin & ~d1[0, 0].isnan()]), r


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, 0.25, -3.7])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
def test_policy_inplace_strides_and_scale(dtype, scale):
    x, y = _logits(3, 6, 264, dtype)
    y = _mask(y)
    adv, old, ref = _policy_inputs(x, y, 1.0, 1)
    _policy_case(x, y, adv, old, ref, 0.1, 1.0, "mean", inplace=False, scale=scale)
    _policy_case(x, y, adv, old, ref, 0.1, 1.0, "mean", inplace=True, scale=scale)
    wide, _ = _logits(3, 6, 300, dtype)
    wide[..., 5:269] = x
    _policy_case(wide, y, adv, old, ref, 0.1, 1.0, "sum", inplace=True, scale=scale, view=lambda t: t[..., 5:269])
    first, _ = _logits(6, 3, 264, dtype)
    first.copy_(x.transpose(0, 1))
    _policy_case(first, y, adv, old, ref, 0.1, 1.0, "sequence", inplace=True, scale=scale,
                 view=lambda t: t.transpose(0, 1))
    one, yy = x[:, :1].contiguous(), y[:, :1]
    _policy_case(one, yy, adv, old[:, :1], ref[:, :1], 0.1, 1.0, "sum", inplace=True, scale=scale)


@pytest.mark.gpu
def test_policy_nothing_kept_and_masked_garbage():
    """Where nothing is kept the loss is 0; NaN in the logits, log-probabilities
    and advantages of ignored tokens reach nothing."""
    from kernels.logprob import forge_policy_loss

    x, y = _logits(2, 5, 100, BF16)
    none = torch.full_like(y, IGNORE)
    adv, old, ref = _policy_inputs(x, y, 1.0, 0, per_token=True)
    for reduction in ("mean", "sequence", "sum"):
        xg = x.cuda().requires_grad_(True)
        o = forge_policy_loss(xg, none.cuda(), adv.cuda(), old.cuda(), ref.cuda(), kl_coef=0.1, reduction=reduction)
        (d,) = torch.autograd.grad(o.loss, xg)
        assert o.loss.item() == 0.0 and (d == 0).all() and (o.logps == 0).all() and (o.kl == 0).all()
    y[0, 1] = y[1, 3] = IGNORE
    a = forge_policy_loss(x.cuda(), y.cuda(), adv.cuda(), old.cuda(), ref.cuda(), kl_coef=0.1)
    for t in (x, adv, old, ref):
        t[0, 1] = t[1, 3] = float("nan")
    xg = x.cuda().requires_grad_(True)
    b = forge_policy_loss(xg, y.cuda(), adv.cuda(), old.cuda(), ref.cuda(), kl_coef=0.1)
    assert torch.equal(a.loss, b.loss) and torch.equal(a.logps, b.logps) and torch.equal(a.kl, b.kl)
    (d,) = torch.autograd.grad(b.loss, xg)
    assert not d.isnan().any()
    empty = torch.zeros(2, 0, 100, device="cuda", requires_grad=True)
    o = forge_policy_loss(empty, torch.zeros(2, 0, device="cuda", dtype=torch.long), torch.ones(2, device="cuda"))
    assert o.loss.item() == 0.0 and torch.autograd.grad(o.loss, empty)[0].shape == empty.shape


@pytest.mark.gpu
def test_policy_backward_runs_once():
    from kernels.logprob import forge_policy_loss

    x, y = _logits(2, 3, 64, FP32)
    xg = x.cuda().requires_grad_(True)
    o = forge_policy_loss(xg, y.cuda(), torch.ones(2).cuda())
    torch.autograd.grad(o.loss, xg, retain_graph=True)
    with pytest.raises(RuntimeError, match="runs once"):
        torch.autograd.grad(o.loss, xg)
    xl = x.cuda().requires_grad_(True) * 1.0
    square = (xl * xl).sum()
    forge_policy_loss(xl, y.cuda(), torch.ones(2).cuda(), inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        square.backward()


@pytest.mark.gpu
def test_results_repeat_bit_for_bit_and_two_calls_at_once():
    """The same call on two streams at once gives the same bits: workspaces are
    a call's own."""
    from kernels.logprob import forge_policy_loss, forge_preference_loss

    x, y = _logits(4, 200, 9000, BF16)
    x, y = x.cuda(), _mask(y).cuda()
    adv, ref = torch.randn(4).cuda(), torch.randn(4).cuda()

    def both():
        xg = x.clone().requires_grad_(True)
        a = forge_policy_loss(xg, y, adv)
        b = forge_preference_loss(xg, y, ref)
        return (a.loss, a.logps, b.loss, b.rewards, *torch.autograd.grad(a.loss, xg), *torch.autograd.grad(b.loss, xg))

    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(both())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(p, q) for p, q in zip(want, g))


@pytest.mark.gpu
def test_graphs():
    """Scoring, a preference step and a policy step captured (two graphs that
    share nothing), replayed with new inputs against eager runs."""
    from kernels.logprob import forge_policy_loss, forge_preference_loss, forge_token_logps

    x, y = _logits(4, 20, 3000, BF16)
    x, y = x.cuda(), _mask(y).cuda()
    adv, ref = torch.randn(4).cuda(), torch.randn(4).cuda()
    leaf = x.clone().requires_grad_(True)

    def preference(t):
        o = forge_preference_loss(t, y, ref, label_smoothing=0.1)
        return (o.loss, o.logps, *torch.autograd.grad(o.loss, t))

    def policy(t):
        with torch.no_grad():
            old = forge_token_logps(t, y)
        o = forge_policy_loss(t, y, adv, old + 0.1, old - 0.2, kl_coef=0.1)
        return (old, o.loss, o.kl, *torch.autograd.grad(o.loss, t))

    graphs, outs = [], []
    for step in (preference, policy):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(leaf)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(leaf))
        graphs.append(g)
    fresh = x.clone().requires_grad_(True)
    for i in range(4):
        x.normal_(0, 2)
        leaf.detach().copy_(x)
        fresh.detach().copy_(x)
        adv.normal_()
        for g, step, out in zip(graphs, (preference, policy), outs):
            g.replay()
            eager = step(fresh)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager)), (i, step.__name__)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Logits of more than 2^31 elements; the last rows against a call of their own."""
    from kernels.logprob import forge_policy_loss

    v, s = 128256, 8400
    n = 2
    x = torch.zeros(n, s, v, device="cuda", dtype=BF16)
    y = torch.full((n, s), IGNORE, device="cuda")
    tail, ty = _logits(1, 3, v, BF16, seed=5)
    x[1, -3:], y[1, -3:] = tail[0].cuda(), ty[0].cuda()
    adv = torch.ones(n, device="cuda")
    xg = x.requires_grad_(True)
    o = forge_policy_loss(xg, y, adv)
    (d,) = torch.autograd.grad(o.loss, xg)
    small = tail.cuda().requires_grad_(True)
    want = forge_policy_loss(small, ty.cuda(), adv[:1])
    (dw,) = torch.autograd.grad(want.loss, small)
    assert (o.logps[1, -3:] - want.logps[0]).abs().max() <= 2 * (64 + v / 8192 + 60) * U
    assert ((d[1, -3:] - dw[0]).abs() <= dw[0].abs() * 2.0 ** -7 + 1e-9).all()
    assert (d[0, -1] == 0).all() and (d[1, -4] == 0).all()
