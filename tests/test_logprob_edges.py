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


# ---------------------------------------------------------------------------
# policy rows at a type's extreme values
# ---------------------------------------------------------------------------
U = 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("temperature", [1e-6, 0.01, 0.35, 0.7, 0.72, 0.73, 1.0, 3.0, 1e6])
@pytest.mark.parametrize("s,v", [(4, 2052), (300, 515), (600, 515), (300, 20003), (300, 65544), (300, 131072)])
def test_policy_rows_at_extreme_values(s, v, temperature, dtype):
    """Rows of the lowest or the largest value, some with a few at the other end.
    fp32 within (64 + V / 8192) U for the sum and the logarithm (the exponents
    are 0 or far below but in fp16 at t = 1e6, where they reach 0.2), 4 U of logp
    for its product with 1 / t and its rounding; a gradient is rounded to its
    type once."""
    from kernels.logprob import forge_policy_loss

    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.zeros(1, s, v, dtype=dtype)
    y = torch.full((1, s), 3)
    x[0, 0] = low
    x[0, 1] = high
    x[0, 2], x[0, 2, 3] = low, 0.5 * high      # the target is the one above
    x[0, 3], x[0, 3, v - 1] = low, high        # the target is not
    if s > 4:
        x[0, 4], x[0, 4, :5] = low, high       # a few share it
        x[0, 5], x[0, 5, v // 2:] = high, low
        x[0, 6], x[0, 6, 9:] = low / 2, low
        x[0, 7] = low / 4
        y[0, 8:] = IGNORE
    n = min(s, 8)
    lp_all = (x[0, :n].double() / temperature).log_softmax(-1)
    lp = lp_all[:, 3]
    hot = torch.zeros_like(lp_all)
    hot[:, 3] = 1.0
    grad = lp_all.exp() - hot

    xg = x.cuda().requires_grad_(True)
    # with an advantage of t a row's gradient is p - onehot
    o = forge_policy_loss(xg, y.cuda(), torch.full((1,), temperature, device="cuda"), temperature=temperature,
                          reduction="sum")
    (got,) = torch.autograd.grad(o.loss, xg)
    assert (o.logps[0, n:] == 0).all() and (got[0, n:] == 0).all()
    e = (64 + v / 8192 + 3 * 0.2) * U
    # equal where a distance / t is past fp32's range
    off = torch.where(o.logps[0, :n].cpu() == lp.float(), 0.0, (o.logps[0, :n].cpu().double() - lp).abs())
    assert (off <= e + lp.abs() * 4 * U).all(), off
    bound = grad.abs() * (torch.finfo(dtype).eps / 2 + 2 * e + 8 * U) + torch.finfo(dtype).smallest_normal
    assert ((got[0, :n].double().cpu() - grad).abs() <= bound).all()
    assert abs(o.loss.item() + temperature * n) <= temperature * n * 4 * U  # r = 1


# ---------------------------------------------------------------------------
# a divergence that is only reported
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("s", [6, 300, 600])
def test_divergence_without_a_weight(s, dtype):
    """ref_logps with kl_coef = 0 report kl and change nothing else, infinite
    as it may be: a token that the reference rules out (-inf), one that the
    policy does, and one that the reference finds e^1000 times likelier."""
    from kernels.logprob import forge_policy_loss

    g = torch.Generator().manual_seed(s)
    inf = float("inf")
    x = torch.randn(1, s, 1000, generator=g).to(dtype)
    y = torch.randint(0, 1000, (1, s), generator=g)
    y[0, 5] = IGNORE
    x[0, 1, y[0, 1]] = -inf
    ref = torch.full((1, s), -7.0)
    ref[0, 0], ref[0, 1], ref[0, 2], ref[0, 5] = -inf, -3.0, 1000.0, float("nan")
    old = torch.full((1, s), -7.5)
    adv = torch.randn(1, s, generator=g)
    xg = x.cuda().requires_grad_(True)

    def call(ref, kl_coef=0.0):
        o = forge_policy_loss(xg, y.cuda(), adv.cuda(), old.cuda(), None if ref is None else ref.cuda(), kl_coef=kl_coef)
        return o, torch.autograd.grad(o.loss, xg)[0]

    want, dw = call(None)
    got, d = call(ref)
    assert want.loss.isfinite() and torch.equal(got.loss, want.loss) and torch.equal(got.logps, want.logps)
    assert torch.equal(d, dw) and d.isfinite().all() and (want.kl == 0).all()
    assert (got.kl[0, :3] == inf).all() and got.kl[0, 3:].isfinite().all() and got.kl[0, 5] == 0
    f = ref[0, 3:5].double() - got.logps[0, 3:5].double().cpu()
    kl = torch.expm1(f) - f
    # logps come back rounded (U of themselves), which moves kl by its slope
    off = (torch.expm1(f).abs() + f.exp() * 1e-6) * got.logps[0, 3:5].double().cpu().abs() * 2.0 ** -23 + kl * 2.0 ** -22
    assert ((got.kl[0, 3:5].double().cpu() - kl).abs() <= off).all()
    with torch.no_grad():
        plain = forge_policy_loss(xg, y.cuda(), adv.cuda(), old.cuda(), ref.cuda())
    assert plain.loss.isfinite() and (plain.kl[0, :3] == inf).all()
    # with a weight the loss is infinite, not NaN; a token that the reference rules out keeps a finite gradient
    weighted, d = call(ref, 0.1)
    assert weighted.loss == inf and d[0, 0].isfinite().all() and torch.equal(weighted.kl, got.kl)


@pytest.mark.gpu
@pytest.mark.parametrize("s", [6, 300, 600])
def test_kl_of_targets_out_of_range(s):
    """NaN where there is a reference, 0 where there is none, whatever the size
    of the batch."""
    from kernels.logprob import forge_policy_loss

    x = torch.randn(1, s, 100).bfloat16().cuda().requires_grad_(True)
    y = torch.randint(0, 100, (1, s)).cuda()
    y[0, 1], y[0, 2] = 100, -5
    ref = torch.full((1, s), -5.0, device="cuda")
    none, some = (forge_policy_loss(x, y, torch.ones(1, device="cuda"), ref_logps=r) for r in (None, ref))
    assert (none.kl == 0).all() and none.loss.isnan() and some.loss.isnan()
    assert some.kl[0, 1:3].isnan().all() and not some.kl[0, 0].isnan() and not some.kl[0, 3:].isnan().any()


# ---------------------------------------------------------------------------
# answers that the policy rules out
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("smoothing,chosen,want", [(0.0, False, 0.0), (0.0, True, float("inf")), (1.0, True, 0.0),
                                                   (0.1, False, float("inf"))])
def test_preference_of_answers_ruled_out(smoothing, chosen, want):
    """A token at -inf makes its answer's log-probability -inf and h infinite:
    the sigmoid loss of that pair is 0 or infinite (a term of weight 0 is left
    out: 0 times infinity is NaN), and the other pair's is its own."""
    from kernels.logprob import forge_preference_loss

    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 3, 40, generator=g)
    y = torch.randint(0, 40, (4, 3), generator=g).cuda()
    xg = x.cuda().requires_grad_(True)
    clean = forge_preference_loss(xg, y, label_smoothing=smoothing, reduction="none")
    x[0 if chosen else 2, 1, y[0 if chosen else 2, 1]] = -float("inf")
    xg = x.cuda().requires_grad_(True)
    o = forge_preference_loss(xg, y, label_smoothing=smoothing, reduction="none")
    assert o.loss[0] == want and torch.equal(o.loss[1], clean.loss[1])
    assert o.logps[0 if chosen else 2] == -float("inf")
    (d,) = torch.autograd.grad(o.loss, xg, torch.ones_like(o.loss))
    assert d.isfinite().all()
    if want == 0.0:
        assert (d[[0, 2]] == 0).all()
        mean = forge_preference_loss(xg, y, label_smoothing=smoothing)
        assert abs(mean.loss.item() - o.loss[1].item() / 2) <= 2.0 ** -23 * o.loss[1].item()


# ---------------------------------------------------------------------------
# masked columns
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,v,temperature", [(3, 30011, 1.0), (40, 128256, 0.7), (700, 1003, 1.0), (1100, 5000, 2.0)])
def test_masked_columns_change_nothing_else(rows, v, temperature, dtype):
    """Scattered columns at -infinity, at the type's lowest value or at -1e4
    have no share: the sums over the others, with the corrections of their
    rounding, are the same bit for bit.  (Targets near probability 1, where a
    log-probability shows its row's sum to 1e-9.)"""
    from kernels.logprob import forge_token_logps

    g = torch.Generator().manual_seed(rows)
    x = torch.randn(1, rows, v, generator=g) * 2
    y = torch.randint(0, v, (1, rows), generator=g)
    x.scatter_(-1, y.unsqueeze(-1), 14.0)
    masked = torch.rand(1, rows, v, generator=g) < 0.1
    masked.scatter_(-1, y.unsqueeze(-1), False)
    results = []
    for value in (-float("inf"), torch.finfo(dtype).min, -1e4):
        xg = x.masked_fill(masked, value).to(dtype).cuda().requires_grad_(True)
        lp = forge_token_logps(xg, y.cuda(), temperature=temperature)
        (d,) = torch.autograd.grad(lp, xg, torch.ones_like(lp))
        assert (d[masked.cuda()] == 0).all()
        results.append((lp.detach(), d))
    want = (x.masked_fill(masked, -float("inf")).to(dtype).double() / temperature).log_softmax(-1)
    want = want.gather(-1, y.unsqueeze(-1)).squeeze(-1)
    assert ((results[0][0].double().cpu() - want).abs() <= (64 + v / 8192 + 3 * 30) * U + want.abs() * U).all()
    for lp, d in results[1:]:
        assert torch.equal(lp, results[0][0]) and torch.equal(d, results[0][1])


# ---------------------------------------------------------------------------
# in place
# ---------------------------------------------------------------------------
def test_inplace_of_a_leafs_view_is_refused():
    """A view of a leaf is the leaf's data, which its gradient may not replace."""
    from kernels.logprob import forge_policy_loss, forge_preference_loss
    from kernels.logprob._rows import check_inplace

    leaf, y = torch.zeros(4, 3, 8, requires_grad=True), torch.zeros(4, 3, dtype=torch.long)
    for view in (leaf, leaf[:], leaf.view(4, 3, 8), leaf[:, :, :5], leaf.transpose(0, 1), leaf[1:].narrow(1, 0, 2),
                 torch.zeros(5, 3, 8)[1:].requires_grad_(True)):
        with pytest.raises(ValueError, match="not a leaf"):
            check_inplace(view)
    with pytest.raises(ValueError, match="not a leaf"):
        forge_policy_loss(leaf[:], y, torch.zeros(4), inplace=True)
    with pytest.raises(ValueError, match="not a leaf"):
        forge_preference_loss(leaf.view(4, 3, 8), y, inplace=True)
    for result in (leaf * 1.0, (leaf * 1.0)[:, 1:], leaf.detach(), leaf.detach()[1:], torch.zeros(2, 3, 8)[:, :2]):
        check_inplace(result)


# ---------------------------------------------------------------------------
# loss scaling
# ---------------------------------------------------------------------------
def _scaled_case(n, s, v, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, s, v, generator=g) * 2).to(dtype)
    y = torch.randint(0, v, (n, s), generator=g)
    y[:, 0] = IGNORE
    return x, y, torch.randn(n, generator=g)


def test_grad_scale_refusals():
    from kernels.logprob import forge_policy_loss

    x, y, adv = _scaled_case(2, 3, 8, torch.float16)
    for bad in (0.0, -1.0, 1e-60, 1e60, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="grad_scale must be positive"):
            forge_policy_loss(x, y, adv, grad_scale=bad)
    with pytest.raises(ValueError, match="one element"):
        forge_policy_loss(x, y, adv, grad_scale=torch.ones(2))
    with pytest.raises(TypeError, match="floating point"):
        forge_policy_loss(x, y, adv, grad_scale=torch.ones(1, dtype=torch.long))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        forge_policy_loss(x, y, adv, grad_scale=torch.ones(()))


@pytest.mark.gpu
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("kind", ["float", "tensor", "scaler"])
@pytest.mark.parametrize("n,s,v", [(8, 1024, 130), (2, 100, 3003), (4, 100, 20000)])
def test_fp16_gradients_under_loss_scaling(n, s, v, kind, inplace):
    """"mean" over the tokens puts a column's gradient far below fp16's least
    (6e-8): with grad_scale what is rounded is the scaled gradient, to half a
    step of fp16 (2^-11) or of its subnormals, over the fp32 error of p (2 e,
    e = (64 + V / 8192 + 3 R) U with R the range of a row of logits, below 40)
    and 8 U of the coefficient's products."""
    from kernels.logprob import forge_policy_loss
    from oracle import logprob as O

    scale = 65536.0
    x, y, adv = _scaled_case(n, s, v, torch.float16)
    leaf = x.cuda().requires_grad_(True)
    scaler = torch.amp.GradScaler("cuda", init_scale=scale)
    given = {"float": scale, "tensor": torch.tensor(scale, device="cuda"), "scaler": scaler.get_scale()}[kind]
    o = forge_policy_loss(leaf * 1.0, y.cuda(), adv.cuda(), grad_scale=given, inplace=inplace)
    up = scaler.scale(o.loss) if kind == "scaler" else o.loss * scale
    (d,) = torch.autograd.grad(up, leaf)
    plain = forge_policy_loss(leaf, y.cuda(), adv.cuda())
    assert torch.equal(plain.loss, o.loss) and torch.equal(plain.logps, o.logps)  # the loss is not scaled
    kept = y != IGNORE
    lp = O.token_logps(x, y)
    _, _, coef = O.policy(lp, kept, adv.unsqueeze(1).expand(n, s), None, None, 0.2, 0.2, 0.0, "mean")
    want = O.dlogits(x, y, coef * scale)
    e = (64 + v / 8192 + 3 * 40) * U
    bound = want.abs() * (2.0 ** -11 + 2 * e + 8 * U) + 2.0 ** -25
    assert ((d.double().cpu() - want).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_grad_scale_other_than_the_incoming_gradient(dtype):
    """What arrives divided by grad_scale multiplies what is stored, which is
    rounded once more; powers of two change nothing but subnormals."""
    from kernels.logprob import forge_policy_loss

    x, y, adv = (t.cuda() for t in _scaled_case(3, 40, 77, dtype))
    x = x.requires_grad_(True)

    def grad(grad_scale, up):
        o = forge_policy_loss(x, y, adv, reduction="sum", grad_scale=grad_scale)
        return torch.autograd.grad(o.loss, x, torch.tensor(up, device="cuda"))[0]

    want = grad(None, 1.0)
    least = torch.finfo(dtype).smallest_normal
    for grad_scale, up in ((16.0, 16.0), (16.0, 1.0), (1.0, 1.0), (1.0, 16.0), (256.0, 4.0)):
        got = grad(grad_scale, up).double() / up
        assert ((got - want.double()).abs() <= least).all(), (grad_scale, up)
    # the scale is the call's own: a buffer that changes afterwards does not count
    s = torch.tensor(8.0, device="cuda")
    o = forge_policy_loss(x, y, adv, reduction="sum", grad_scale=s)
    s.mul_(2.0)
    (got,) = torch.autograd.grad(o.loss, x, torch.tensor(8.0, device="cuda"))
    assert ((got.double() / 8 - want.double()).abs() <= least).all()
