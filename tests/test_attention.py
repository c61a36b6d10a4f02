"""Attention over packed sequences and dense batches (`forge_varlen_attention`,
`forge_attention`).

Tolerances are derived in oracle/attention.py, before the first run: scores,
statistics and sums in fp32, and one rounding to the 16-bit type (half a step:
finfo.eps / 2 relative, half the spacing of its subnormals absolute) of each
probability, each gradient of a score, and each result."""
import math

import pytest
import torch

from oracle.attention import head_fwd_bwd, packed_fwd_bwd

BF16, FP16 = torch.bfloat16, torch.float16


def _unit(dtype):
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _make(lens_q, lens_k, H, kv, D, dtype, seed=0, tail_q=0, tail_k=0, layout="plain", std=1.0):
    g = torch.Generator().manual_seed(seed)
    T, Tk = sum(lens_q) + tail_q, sum(lens_k) + tail_k
    if layout == "packed":  # columns of one projection's output
        assert T == Tk
        t = (torch.randn(T, H + 2 * kv, D, generator=g) * std).to(dtype)
        q, k, v = t.split([H, kv, kv], 1)
    elif layout == "heads":  # tokens of a head beside each other
        q, k, v = ((torch.randn(h, n, D, generator=g) * std).to(dtype).transpose(0, 1)
                   for h, n in ((H, T), (kv, Tk), (kv, Tk)))
    else:
        q, k, v = ((torch.randn(n, h, D, generator=g) * std).to(dtype) for h, n in ((H, T), (kv, Tk), (kv, Tk)))
    do = torch.randn(T, H, D, generator=g).to(dtype)
    return q, k, v, do


def _within(got, ref, err, what):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, what
    inf = torch.isinf(ref)
    assert torch.equal(torch.isinf(got), inf), what
    over = ((got - ref).abs() - err)[~inf]
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, f"{what}: off by {worst:.3e} more than the bound"


def _check(lens_q, lens_k, H, kv, D, dtype, causal=True, train=True, scale=None, **kw):
    from kernels.attention import forge_varlen_attention

    q, k, v, do = _make(lens_q, lens_k, H, kv, D, dtype, **kw)
    cu_q, cu_k = _offsets(lens_q), _offsets(lens_k)
    ref = packed_fwd_bwd(q, k, v, do, cu_q, cu_k, scale or D ** -0.5, causal, *_unit(dtype))

    def gpu(t):  # keeps the strides
        base = t._base if t._base is not None else t
        return torch.as_strided(base.cuda(), t.shape, t.stride(), t.storage_offset())

    qg, kg, vg = (gpu(t).detach().requires_grad_(train) for t in (q, k, v))
    out, lse = forge_varlen_attention(qg, kg, vg, torch.tensor(cu_q, device="cuda", dtype=torch.int32),
                                      torch.tensor(cu_k, device="cuda", dtype=torch.int32), causal=causal, scale=scale,
                                      return_lse=True)
    assert out.dtype == dtype and lse.dtype == torch.float32
    _within(out, ref.o, ref.o_err, "out")
    _within(lse, ref.lse, ref.lse_err, "lse")
    if train:
        for n, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (qg, kg, vg), do.cuda())):
            _within(x, getattr(ref, n), getattr(ref, n + "_err"), n)


# ---------------------------------------------------------------------------
# the oracle and refusals (CPU)
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n,m,causal", [(5, 5, True), (3, 7, True), (7, 3, True), (4, 6, False), (1, 1, True)])
def test_oracle_against_autograd_and_differences(n, m, causal):
    g = torch.Generator().manual_seed(n * 10 + m)
    q, k, v, do = (torch.randn(r, 8, generator=g, dtype=torch.float64) for r in (n, m, m, n))
    r = head_fwd_bwd(q, k, v, do, 0.3, causal, 0.0, 0.0)

    def f(q, k, v):
        s = 0.3 * q @ k.T
        if causal:
            s = s.masked_fill(~torch.ones(n, m, dtype=torch.bool).tril(m - n), float("-inf"))
        p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
        return p @ v

    torch.testing.assert_close(r.o, f(q, k, v))
    assert torch.equal(torch.isinf(r.lse), torch.tensor([causal and i + m - n < 0 for i in range(n)]))
    step = 1e-6
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        num = torch.zeros_like(x)
        for i in range(x.numel()):
            e = torch.zeros_like(x).view(-1)
            e[i] = step
            e = e.view_as(x)
            args = {"dq": q, "dk": k, "dv": v}
            hi, lo = ((f(*[t + s * e if key == name else t for key, t in args.items()]) * do).sum() for s in (1, -1))
            num.view(-1)[i] = (hi - lo) / (2 * step)
        torch.testing.assert_close(getattr(r, name), num, rtol=1e-6, atol=1e-7)


def test_refusals():
    from kernels.attention import forge_attention, forge_varlen_attention

    cu = torch.tensor([0, 4], dtype=torch.int32)

    def call(q=(4, 4, 64), k=(4, 2, 64), v=None, dtype=BF16, cu=cu, **kw):
        return forge_varlen_attention(torch.zeros(q, dtype=dtype), torch.zeros(k, dtype=dtype),
                                      torch.zeros(v or k, dtype=kw.pop("v_dtype", dtype)), cu, **kw)

    for match, kw in (("dimensions", {"q": (4, 64)}), ("same shape", {"v": (4, 1, 64)}), ("head_dim", {"k": (4, 2, 32)}),
                      ("multiple of 8", {"q": (4, 4, 20), "k": (4, 2, 20)}),
                      ("multiple of 8", {"q": (4, 4, 264), "k": (4, 2, 264)}),
                      ("divides", {"k": (4, 3, 64)}), ("positive", {"scale": 0.0}), ("positive", {"scale": float("nan")}),
                      ("positive", {"scale": float("inf")}), ("positive", {"scale": -1.0})):
        with pytest.raises(ValueError, match=match):
            call(**kw)
    with pytest.raises(TypeError, match="fp16 or bf16"):
        call(dtype=torch.float32)
    with pytest.raises(TypeError, match="same dtype"):
        call(v_dtype=FP16)
    with pytest.raises(RuntimeError, match="GPU"):
        call()
    with pytest.raises(ValueError, match="batch"):
        forge_attention(*(torch.zeros(b, 2, 4, 64, dtype=BF16) for b in (1, 2, 2)))


def test_entry_point_refusals():
    from forge_hip import _lib as L

    rows = [16, 0, 512, 64]

    def fwd(dtype=2, q=rows, k=rows, v=rows, o=rows, cu=(16, 16), sizes=(1, 4, 4, 4, 2, 64), scale=0.1, low=None):
        return L.forge_attention_fwd(dtype, *q, *k, *v, *o, None, low, *cu, *sizes, scale, 1, None, None)

    assert fwd(dtype=0) == 2 and b"dtype" in L.forge_last_error()
    assert fwd(sizes=(1, 4, 4, 4, 2, 60)) == 2 and b"head_dim" in L.forge_last_error()
    assert fwd(sizes=(1, 4, 4, 4, 2, 512)) == 2
    assert fwd(sizes=(1, 4, 4, 4, 3, 64)) == 1 and b"heads" in L.forge_last_error()
    assert fwd(sizes=(-1, 4, 4, 4, 2, 64)) == 1
    assert fwd(sizes=(1, -4, 4, 4, 2, 64)) == 1
    assert fwd(sizes=(1, 1 << 40, 4, 4, 2, 64)) == 1
    assert fwd(cu=(None, 16)) == 1 and b"one side" in L.forge_last_error()
    assert fwd(scale=0.0) == 1 and fwd(scale=float("nan")) == 1
    for name, at in (("q", "q"), ("k", "k"), ("v", "v"), ("out", "o")):
        assert fwd(**{at: [None, 0, 512, 64]}) == 1 and f"{name} is NULL".encode() in L.forge_last_error()
        assert fwd(**{at: [24, 0, 512, 64]}) == 1 and b"aligned" in L.forge_last_error()
        assert fwd(**{at: [16, 0, 516, 64]}) == 1
        assert fwd(**{at: [16, 0, 1 << 23, 64]}) == 1 and b"stride" in L.forge_last_error()
    # 2049 keys of one sequence are read in chunks
    assert L.forge_attention_fwd_workspace(1, 1, 1, 2049, 4, 2, 64) == (2049 // 128 + 1) * 4 * 66 * 4
    long = (1, 1, 2049, 4, 2, 64)
    args = [2, *rows, *rows, *rows, *rows, None, None, 16, 16, *long, 0.1, 1]
    assert L.forge_attention_fwd(*args, None, None) == 1 and L.forge_attention_fwd(*args, 24, None) == 1
    assert b"work" in L.forge_last_error()
    assert fwd(low=24) == 1 and b"low" in L.forge_last_error()

    def bwd(dtype=2, lse=16, low=16, work=16):
        return L.forge_attention_bwd(dtype, *(rows * 5), lse, low, *(rows * 3), 16, 16, 1, 4, 4, 4, 2, 64, 0.1, 1, work, None)

    assert bwd(lse=None) == 1 and bwd(low=None) == 1 and b"lse, low or work" in L.forge_last_error()
    assert bwd(work=None) == 1 and bwd(work=24) == 1
    assert bwd(dtype=0) == 2 and bwd(low=24) == 1 and b"low" in L.forge_last_error()
    assert L.forge_attention_bwd_workspace(1, 1, 4, 4, 4, 2, 64) == 4 * 4 * 2 * 4
    # few keys, many heads: 16 parts of 300 keys
    assert L.forge_attention_bwd_workspace(0, 1, 300, 300, 16, 1, 64) == 300 * 16 * 2 * 4 + 16 * 300 * 2 * 64 * 4
    assert L.forge_attention_bwd_workspace(1, 1, 4, 4, 4, 3, 64) == -1
    assert L.forge_attention_fwd_workspace(1, 1, 4, 4, 4, 3, 64) == -1
    # nothing to do
    empty = [None, 0, 0, 0]
    assert fwd(q=empty, o=empty, sizes=(1, 0, 4, 4, 2, 64)) == 0


# ---------------------------------------------------------------------------
# kernels
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("H,kv,D", [(4, 2, 128), (2, 2, 64), (7, 1, 96), (4, 4, 8), (3, 1, 256), (2, 1, 200), (16, 8, 40)])
def test_packed_sequences(H, kv, D, dtype):
    lens = [1, 130, 64, 0, 257, 31]
    _check(lens, lens, H, kv, D, dtype, layout="packed")


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens_q,lens_k", [([5], [700]), ([200, 3], [264, 3]), ([300, 40], [100, 40]), ([129, 7], [0, 65]),
                                           ([64], [64]), ([128, 128], [128, 192]), ([1] * 70, list(range(70)))])
def test_lengths(lens_q, lens_k, causal):
    """Keys before the queries, fewer keys than queries, none, whole tiles, more sequences than lanes."""
    _check(lens_q, lens_k, 4, 2, 64, BF16, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,H,kv,D", [(BF16, 32, 8, 128), (FP16, 8, 8, 64), (BF16, 16, 1, 256), (FP16, 14, 2, 72)])
@pytest.mark.parametrize("lens_q,lens_k", [([1, 1, 1], [1000, 1, 129]), ([1, 0, 2, 1], [0, 5, 2049, 128]), ([3], [300]),
                                           ([0, 4, 0, 0], [50, 2, 0, 33])])
def test_few_queries(dtype, H, kv, D, lens_q, lens_k):
    """One token a sequence and a few: the kernel that cuts the keys into chunks."""
    _check(lens_q, lens_k, H, kv, D, dtype, train=False)


@pytest.mark.gpu
def test_few_queries_with_gradients_and_without_causality():
    _check([1, 2], [500, 40], 8, 2, 64, BF16)
    _check([1, 2], [500, 40], 8, 2, 64, BF16, causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("lens_q", [[70, 20], [1, 1]])
def test_rows_outside_the_sequences_are_zeros(lens_q):
    _check(lens_q, [90, 40], 4, 2, 64, BF16, tail_q=9, tail_k=150)


@pytest.mark.gpu
@pytest.mark.parametrize("std,scale", [(6.0, None), (1.0, 3.0), (1.0, 1e-4), (30.0, None)])
def test_sharp_and_flat_scores(std, scale):
    _check([150, 33], [150, 33], 2, 1, 64, FP16, std=std, scale=scale)
    _check([150, 1], [150, 300], 2, 1, 128, BF16, std=std, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("D,kv", [(64, 2), (128, 1), (256, 4)])
@pytest.mark.parametrize("size", [2.0 ** -10, 2.0 ** 9])
def test_gradients_of_fp16_over_its_range(size, D, kv):
    """Small gradients: p and ds are held as multiples (2^-14 of the type's smallest steps).  Large ones, where
    those multiples would pass its largest value (|do . v| over 2^13): as they come."""
    from kernels.attention import forge_varlen_attention

    lens = [300, 1, 77]
    q, k, v, do = _make(lens, lens, 4, kv, D, FP16)
    do = (do * size).half()
    at = _offsets(lens)
    unit, tiny = _unit(FP16)
    ref = packed_fwd_bwd(q, k, v, do, at, at, D ** -0.5, True, unit, tiny, tiny * 2.0 ** -14 if size < 1 else tiny)
    assert ref.dq.abs().max() < 60000
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    cu = torch.tensor(at, device="cuda", dtype=torch.int32)
    grads = torch.autograd.grad(forge_varlen_attention(*leaves, cu, cu), leaves, do.cuda())
    for n, x in zip(("dq", "dk", "dv"), grads):
        _within(x, getattr(ref, n), getattr(ref, n + "_err"), n)


@pytest.mark.gpu
def test_tokens_of_a_head_beside_each_other():
    _check([90, 40], [90, 40], 4, 2, 64, BF16, layout="heads")


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,kv,S,Sk,D", [(2, 4, 2, 130, 130, 128), (3, 2, 1, 1, 200, 64), (2, 4, 4, 70, 200, 64)])
@pytest.mark.parametrize("memory", ["bshd", "bhsd", "odd"])
def test_dense_batches(B, H, kv, S, Sk, D, memory):
    from kernels.attention import forge_attention

    g = torch.Generator().manual_seed(1)

    def make(h, s):
        if memory == "bshd":
            return torch.randn(B, s, h, D, generator=g).to(BF16).cuda().transpose(1, 2)
        if memory == "bhsd":
            return torch.randn(B, h, s, D, generator=g).to(BF16).cuda()
        return torch.randn(B * h * s * D + 1, generator=g).to(BF16).cuda()[1:].view(B, h, s, D)  # unaligned rows

    q, k, v = (make(h, s).requires_grad_(True) for h, s in ((H, S), (kv, Sk), (kv, Sk)))
    out, lse = forge_attention(q, k, v, return_lse=True)
    do = torch.randn(B, H, S, D, generator=g).to(BF16).cuda()
    grads = torch.autograd.grad(out, (q, k, v), do)
    flat = [t.detach().cpu().transpose(1, 2).reshape(-1, t.shape[1], D) for t in (q, k, v, do)]
    ref = packed_fwd_bwd(*flat, _offsets([S] * B), _offsets([Sk] * B), D ** -0.5, True, *_unit(BF16))
    _within(lse.reshape(B * S, H), ref.lse, ref.lse_err, "lse")
    for n, x in zip(("o", "dq", "dk", "dv"), (out, *grads)):
        _within(x.transpose(1, 2).reshape(-1, x.shape[1], D), getattr(ref, n), getattr(ref, n + "_err"), n)


@pytest.mark.gpu
def test_nothing_to_do():
    from kernels.attention import forge_attention, forge_varlen_attention

    z = torch.zeros(0, 2, 64, dtype=BF16, device="cuda", requires_grad=True)
    k = torch.ones(5, 2, 64, dtype=BF16, device="cuda", requires_grad=True)
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    out = forge_varlen_attention(z, k, k, cu, torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda"))
    assert out.shape == z.shape
    (g,) = torch.autograd.grad(out, k, torch.zeros_like(out))
    assert torch.equal(g, torch.zeros_like(k))
    q = torch.ones(5, 2, 64, dtype=BF16, device="cuda", requires_grad=True)
    out, lse = forge_varlen_attention(q, z, z, torch.tensor([0, 2, 5], device="cuda"), cu, return_lse=True)
    assert torch.equal(out, torch.zeros_like(q)) and bool((lse == -math.inf).all())
    assert torch.equal(torch.autograd.grad(out, q, torch.ones_like(q))[0], torch.zeros_like(q))
    # no sequences at all
    out = forge_varlen_attention(q, k, k, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert torch.equal(out, torch.zeros_like(q))
    e = torch.zeros(2, 2, 3, 64, dtype=BF16, device="cuda")
    assert forge_attention(e, e[:, :, :0], e[:, :, :0]).abs().max() == 0
    assert forge_attention(e[:0], e[:0], e[:0]).shape == (0, 2, 3, 64)


@pytest.mark.gpu
def test_offsets_are_checked_when_asked():
    from kernels.attention import forge_varlen_attention

    q = torch.ones(5, 2, 64, dtype=BF16, device="cuda")
    for bad in ([1, 5], [0, 6], [0, 3, 2], [0, -1]):
        with pytest.raises(ValueError, match="begin at 0"):
            forge_varlen_attention(q, q, q, torch.tensor(bad, device="cuda"), validate_offsets=True)
    with pytest.raises(ValueError, match="sequences"):
        forge_varlen_attention(q, q, q, torch.tensor([0, 5], device="cuda"), torch.tensor([0, 2, 5], device="cuda"))
    with pytest.raises(ValueError, match="cu_seqlens_k"):
        forge_varlen_attention(q, q[:3], q[:3], torch.tensor([0, 5], device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("train", [False, True])
def test_many_sequences(train):
    """More than a workgroup looks at in one step (256), of 0 to 3 tokens, one long among them."""
    lens = [i % 4 for i in range(600)]
    lens[300] = 200
    _check(lens, lens, 2, 1, 64, BF16, train=train)


@pytest.mark.gpu
def test_more_tiles_than_one_level_holds():
    _check([700, 1, 300], [700, 1, 300], 3, 1, 64, BF16)
    _check([1, 1500], [1, 1500], 1, 1, 8, FP16)


@pytest.mark.gpu
@pytest.mark.parametrize("queries", [1, 300])
def test_offsets_past_32_bits(queries):
    """A cache whose last sequence begins 2^31 elements from its first: the same bits as from a small one."""
    from kernels.attention import forge_varlen_attention

    row = 4096  # elements from token to token: a layer's slice of a wider cache
    tokens = (1 << 31) // row + 700
    cache = torch.empty(tokens, row, device="cuda", dtype=BF16)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(500, 2, 64, generator=g).to(BF16).cuda() for _ in range(2))
    q = torch.randn(queries, 4, 64, generator=g).to(BF16).cuda()
    kc, vc = (cache[:, i * 128:(i + 1) * 128].view(tokens, 2, 64) for i in (0, 1))
    at = tokens - 600
    kc[at:at + 500], vc[at:at + 500] = k, v
    cu_q = torch.tensor([0, 0, queries], device="cuda", dtype=torch.int32)
    far = forge_varlen_attention(q, kc, vc, cu_q, torch.tensor([0, at, at + 500], device="cuda", dtype=torch.int32))
    near = forge_varlen_attention(q, k, v, cu_q, torch.tensor([0, 0, 500], device="cuda", dtype=torch.int32))
    if queries > 1:
        assert torch.equal(far, near)
    else:  # (a token's keys are cut by the number of all the cache's keys: other sums)
        assert (far.float() - near.float()).abs().max() <= 2.0 ** -7 * v.float().abs().max()


def _special(t, rows, values):
    """t with values at some columns of the rows."""
    t = t.clone()
    for n, row in enumerate(rows):
        for j, x in enumerate(values):
            t[row, n % t.shape[1], (11 * j + 5 * n) % t.shape[2]] = x
    return t


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("H,kv,D", [(2, 1, 64), (4, 2, 128), (2, 2, 256), (3, 1, 40)])
@pytest.mark.parametrize("lens_q,lens_k", [([200, 90], [200, 90]), ([3, 7], [330, 40]), ([100], [300])])
@pytest.mark.parametrize("train", [False, True])
def test_values_that_are_not_finite_where_they_are_not_seen(lens_q, lens_k, H, kv, D, dtype, train):
    """NaN and infinities in keys and values: the queries that do not see them are as they are without."""
    from kernels.attention import forge_varlen_attention

    q, k, v, do = _make(lens_q, lens_k, H, kv, D, dtype)
    at_q, at_k = _offsets(lens_q), _offsets(lens_k)
    # of the first sequence: from its key `first` on, next to the last queries' borders
    first = lens_k[0] - lens_q[0] + lens_q[0] // 2
    rows = list(range(first, lens_k[0], 2))
    inf, nan = float("inf"), float("nan")
    cu_q, cu_k = (torch.tensor(x, device="cuda", dtype=torch.int32) for x in (at_q, at_k))

    def run(k, v):
        leaves = [t.cuda().requires_grad_(train) for t in (q, k, v)]
        out, lse = forge_varlen_attention(*leaves, cu_q, cu_k, return_lse=True)
        return [out.detach(), lse.detach(), *(torch.autograd.grad(out, leaves, do.cuda())[:1] if train else ())]

    plain = run(k, v)
    clean = [i for i in range(at_q[-1]) if not lens_q[0] // 2 <= i < lens_q[0]]
    for bad_k, bad_v in ((k, _special(v, rows, [nan, inf, -inf])), (_special(k, rows, [nan]), _special(v, rows, [nan])),
                         (_special(k, rows, [inf, -inf]), v)):
        for a, b in zip(run(bad_k, bad_v), plain):
            assert torch.equal(a[clean], b[clean])
    # where they are seen: infinities of a value in the columns that have them, with their sign
    out = run(k, _special(v, rows[:1], [inf, -inf]))[0].double().cpu()
    seen = slice(lens_q[0] // 2, lens_q[0])
    want = [head_fwd_bwd(q[:at_q[1], h], k[:at_k[1], h * kv // H], _special(v, rows[:1], [inf, -inf])[:at_k[1], h * kv // H],
                         do[:at_q[1], h], D ** -0.5, True, *_unit(dtype)).o for h in range(H)]
    for h in range(H):
        for x in (inf, -inf):
            hit = want[h][seen] == x
            assert torch.equal(out[seen, h] == x, hit) and (h * kv // H > 0 or hit.any())
    # and a NaN of a key makes all of a query that sees it NaN
    assert run(_special(k, rows[:1], [nan]), v)[0][seen][:, :H // kv].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("lens_q,lens_k", [([600], [600]), ([300, 0, 5, 400], [300, 9, 0, 700])])
@pytest.mark.parametrize("H,kv,D,dtype", [(16, 1, 64, FP16), (12, 2, 128, BF16), (7, 1, 256, BF16), (40, 1, 8, BF16)])
def test_few_keys_and_many_heads(lens_q, lens_k, H, kv, D, dtype):
    """Gradients of keys whose heads go to several workgroups (heads that the parts do not divide)."""
    _check(lens_q, lens_k, H, kv, D, dtype, tail_q=3, tail_k=40)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_few_tokens_with_gradients_over_many_chunks(dtype):
    """Long caches, whose chunks are joined, then trained through: 1 and 2 tokens, none, of 3000 keys and less."""
    _check([1, 2, 0, 1], [3000, 1, 5, 700], 8, 2, 128, dtype, tail_q=1)


@pytest.mark.gpu
@pytest.mark.parametrize("train", [False, True])
def test_one_long_sequence_among_empty_ones(train):
    """As many tokens as few a sequence would be, all of one sequence."""
    lens = [0] * 40 + [150] + [0] * 39
    _check(lens, lens, 4, 2, 64, BF16, train=train)


@pytest.mark.gpu
def test_expanded_keys_and_one_tensor_for_all():
    """One key head expanded to four (stride 0), and q = k = v: gradients add up."""
    from kernels.attention import forge_varlen_attention

    g = torch.Generator().manual_seed(0)
    q, one = torch.randn(90, 4, 64, generator=g).to(BF16), torch.randn(90, 1, 64, generator=g).to(BF16)
    do = torch.randn(90, 4, 64, generator=g).to(BF16).cuda()
    cu = torch.tensor([0, 50, 90], device="cuda", dtype=torch.int32)
    qg, kg = q.cuda().requires_grad_(True), one.cuda().requires_grad_(True)
    out = forge_varlen_attention(qg, kg.expand(-1, 4, -1), kg.expand(-1, 4, -1), cu)
    want = forge_varlen_attention(qg, kg.repeat(1, 4, 1), kg.repeat(1, 4, 1), cu)
    assert torch.equal(out, want)
    for a, b in zip(torch.autograd.grad(out, (qg, kg), do), torch.autograd.grad(want, (qg, kg), do)):
        assert (a.float() - b.float()).abs().max() <= 0.02 * b.float().abs().max()  # (8 roundings of parts as they are added)
    same = q.cuda().requires_grad_(True)
    (a,) = torch.autograd.grad(forge_varlen_attention(same, same, same, cu), same, do)
    leaves = [q.cuda().requires_grad_(True) for _ in range(3)]
    parts = torch.autograd.grad(forge_varlen_attention(*leaves, cu), leaves, do)
    assert (a.float() - sum(p.float() for p in parts)).abs().max() <= 0.02 * a.float().abs().max()


@pytest.mark.gpu
def test_captured_gradients_of_few_keys():
    """The pass whose heads go to several workgroups and are joined, captured and replayed with other values and
    other lengths of the same total, an eager pass between: the same bits."""
    from kernels.attention import forge_varlen_attention

    g = torch.Generator().manual_seed(0)
    q = torch.randn(600, 16, 64, generator=g).to(FP16).cuda().requires_grad_(True)
    k, v = (torch.randn(600, 1, 64, generator=g).to(FP16).cuda().requires_grad_(True) for _ in range(2))
    do = torch.randn(600, 16, 64, generator=g).to(FP16).cuda()
    cu = torch.tensor([0, 200, 600], device="cuda", dtype=torch.int32)

    def step():
        out = forge_varlen_attention(q, k, v, cu)
        grads = torch.autograd.grad(out, (q, k, v), do)
        return (out.detach(), *grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i, at in enumerate(([0, 200, 600], [0, 1, 600], [0, 600, 600], [0, 300, 500])):
        with torch.no_grad():
            cu.copy_(torch.tensor(at, dtype=torch.int32))
            for t in (q, k, v, do):
                t.copy_(torch.randn(t.shape, generator=g).to(FP16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in static]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), f"replay {i}"
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("where", [0, -1])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries", [1, 8, 300])
@pytest.mark.parametrize("keys,above", [(16384, 17.4), (16384, 19.0), (3000, 16.9)])
def test_many_small_probabilities_in_fp16(keys, above, queries, causal, where):
    """One key far above all others, whose probabilities (2^-24 to 2^-27 of its) are below fp16's smallest steps, and
    whose sum is the result.  Each is off by 2^-34 of the largest at most (held 2^9 times as large, half a step of
    2^-24), by its rounding (2^-11 of it) and by that of the result."""
    from kernels.attention import forge_varlen_attention

    k, v = torch.zeros(keys, 1, 64, dtype=FP16), torch.ones(keys, 1, 64, dtype=FP16)
    k[where, 0, 0], v[where] = above, 0
    q = torch.zeros(queries, 2, 64, dtype=FP16)
    q[:, :, 0] = 1
    cu_q, cu_k = (torch.tensor([0, n], device="cuda", dtype=torch.int32) for n in (queries, keys))
    out = forge_varlen_attention(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_k, scale=1.0, causal=causal).double().cpu()
    for i in range(queries):
        sees = keys - queries + i + 1 if causal else keys
        s = k[:sees, 0, 0].double()
        ref = torch.softmax(s, 0) @ v[:sees, 0].double()
        err = ref * 2 * 2.0 ** -11 * (1 + 2.0 ** -8) + sees * 2.0 ** -34 + 2.0 ** -25
        assert bool(((out[i] - ref).abs() <= err).all()), (i, out[i, 0, 0].item(), ref[0].item())


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e36, 8e37])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens_q,lens_k", [([1, 1], [3000, 40]), ([3], [900]), ([200, 5], [200, 1300])])
def test_values_near_the_largest(lens_q, lens_k, causal, size):
    """Sums of probabilities times values pass fp32's range before they are divided by the probabilities' sum; the
    results do not.  Small values beside them keep their accuracy, and keys that are not finite stay apart."""
    from kernels.attention import forge_varlen_attention

    q, k, v, do = _make(lens_q, lens_k, 4, 2, 72, BF16)
    v = (v.float().clamp(-4, 4) * size).to(BF16)
    v[:, :, 1] = (v[:, :, 1].float() * (1e-20 / size)).to(BF16)
    v[:, :, 2] = v[:, :, 2].abs()
    at_q, at_k = _offsets(lens_q), _offsets(lens_k)
    unit, tiny = _unit(BF16)
    ref = packed_fwd_bwd(q, k, v, do * 0, at_q, at_k, 72 ** -0.5, causal, unit, tiny)
    cu_q, cu_k = (torch.tensor(a, device="cuda", dtype=torch.int32) for a in (at_q, at_k))
    out, lse = forge_varlen_attention(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_k, causal=causal, return_lse=True)
    # (a result's error is a share of its own column's terms: the bound of each is made of |v| of that column)
    _within(out, ref.o, ref.o_err, "out")
    _within(lse, ref.lse, ref.lse_err, "lse")
    if causal and lens_q[0] > 3:
        bad = _special(v, list(range(100, 200, 2)), [float("nan"), float("inf")])
        got = forge_varlen_attention(q.cuda(), k.cuda(), bad.cuda(), cu_q, cu_k)
        _within(got[:100], ref.o[:100], ref.o_err[:100], "rows that do not see them")
        assert bool(got[103:200].isnan().any(-1).all()) and bool(got[200:].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens_q,lens_k,row", [([1, 1], [40, 9], 0), ([1, 2], [5000, 30], 0), ([2, 1], [300, 70], 1),
                                               ([200, 60], [200, 60], 37), ([100, 30], [60, 30], 90)])
def test_scores_that_are_all_minus_infinity(lens_q, lens_k, row, causal, dtype):
    """A query that sees keys, all with a score of -inf, has no probabilities: NaN, as in the softmax of its row, and so
    are the gradients that it takes part in.  One that sees no key has zeros."""
    from kernels.attention import forge_varlen_attention

    q, k, v, do = _make(lens_q, lens_k, 4, 2, 64, dtype)
    k[:, :, 0] = 1
    q[:, :, 0] = 0
    bad = q.clone()
    bad[row, 1, 0] = float("-inf")
    cu_q, cu_k = (torch.tensor(_offsets(n), device="cuda", dtype=torch.int32) for n in (lens_q, lens_k))

    def run(q):
        leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
        out, lse = forge_varlen_attention(*leaves, cu_q, cu_k, causal=causal, return_lse=True)
        return [t.detach() for t in (out, lse, *torch.autograd.grad(out, leaves, do.cuda()))]

    (out, lse, dq, dk, dv), plain = run(bad), run(q)
    assert bool(out[row, 1].isnan().all()) and lse[row, 1] == -math.inf and bool(dq[row, 1].isnan().all())
    sees = row + lens_k[0] - lens_q[0] + 1 if causal else lens_k[0]
    assert bool(dk[:sees, 0].isnan().all()) and bool(dv[:sees, 0].isnan().all())
    others = torch.ones(sum(lens_q), 4, dtype=torch.bool)
    others[row, 1] = False
    for a, b in zip((out, lse, dq), plain):
        assert torch.equal(a[others], b[others])
    for a, b in zip((dk, dv), plain[3:]):
        assert torch.equal(a[:, 1], b[:, 1]) and torch.equal(a[lens_k[0]:], b[lens_k[0]:])
    none = [i for i in range(lens_q[0]) if causal and i + lens_k[0] - lens_q[0] < 0]
    assert bool((out[none] == 0).all()) and bool((lse[none] == -math.inf).all()) and bool((dq[none] == 0).all())
    # the definition's, in float64
    s = bad[row, 1].double() @ k[:sees, 0].double().T
    assert bool((s == -math.inf).all()) and bool(torch.softmax(s, 0).isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("H,kv,D", [(2, 1, 64), (4, 2, 128), (2, 2, 256), (3, 1, 40), (16, 1, 64)])
@pytest.mark.parametrize("lens_q,lens_k,row", [([300, 90], [300, 90], 100), ([3, 7], [330, 40], 1), ([100, 40], [60, 40], 45),
                                               ([100, 40], [60, 40], 20), ([70], [500], 33)])
def test_queries_and_gradients_that_are_not_finite(lens_q, lens_k, row, H, kv, D, dtype):
    """NaN and infinities in a query or in the gradient of an output: the gradients of the keys and values that it does
    not see are as they are without, bit by bit, and so are the other queries'."""
    from kernels.attention import forge_varlen_attention

    q, k, v, do = _make(lens_q, lens_k, H, kv, D, dtype)
    cu_q, cu_k = (torch.tensor(_offsets(n), device="cuda", dtype=torch.int32) for n in (lens_q, lens_k))
    inf, nan = float("inf"), float("nan")

    def run(q, do):
        leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
        out = forge_varlen_attention(*leaves, cu_q, cu_k)
        return torch.autograd.grad(out, leaves, do.cuda())

    sees = max(0, row + lens_k[0] - lens_q[0] + 1)  # keys that the row's query sees
    plain = run(q, do)
    for values in ([nan], [inf], [-inf, nan, inf]):
        head = 0
        for bad in (run(_special(q, [row], values), do), run(q, _special(do, [row], values)),
                    run(_special(q, [row], values), _special(do, [row], values))):
            assert torch.equal(bad[0][:row], plain[0][:row]) and torch.equal(bad[0][row + 1:], plain[0][row + 1:])
            for a, b in zip(bad[1:], plain[1:]):
                assert torch.equal(a[sees:], b[sees:]) and torch.equal(a[:, 1:], b[:, 1:])
            if sees:  # and where it is seen, nothing is hidden
                assert not bool(bad[1][:sees, head].isfinite().all(-1).any())
    # a value's gradient: p times the infinity, in its column alone
    dv = run(q, _special(do, [row], [inf]))[2]
    want = plain[2].clone()
    want[:sees, 0, 0] = inf
    assert torch.equal(dv, want)


def _spacing(r, dtype):
    """The spacing of the type's values at r (of the smallest at 0)."""
    e = torch.where(r == 0, 0.0, torch.ldexp(torch.ones_like(r), torch.frexp(r).exponent - 1))
    return e.clamp(min=2.0 ** -14) * 2.0 ** -10 if dtype == FP16 else e.clamp(min=2.0 ** -100) * 2.0 ** -7


# what writes an output: the tiles' kernel, that of few tokens, and the join of its chunks
_WRITERS = [([70, 5], [70, 130]), ([1, 2], [100, 17]), ([1, 2], [300, 8])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 40, 128, 200, 256])
@pytest.mark.parametrize("lens_q,lens_k", _WRITERS)
@pytest.mark.parametrize("size", [1.0, 2.0 ** -15, 300.0])
def test_what_the_rounding_of_an_output_took(size, lens_q, lens_k, D, dtype):
    """The byte a value that the gradients' delta is formed with, in 254ths of a step: with it an output is that of
    exact arithmetic to half of such a part and the fp32 sums' roundings.  Scores of 0, so that all probabilities are
    one power of two and are not rounded; fp16's subnormals among the outputs."""
    from kernels.attention.attention import _forward, _Layout

    _, k, v, _ = _make(lens_q, lens_k, 4, 2, D, dtype)
    v = (v.float() * size).to(dtype)
    q = torch.zeros(sum(lens_q), 4, D, dtype=dtype)
    at_q, at_k = _offsets(lens_q), _offsets(lens_k)
    cu_q, cu_k = (torch.tensor(a, device="cuda", dtype=torch.int32) for a in (at_q, at_k))
    out, _, low = _forward(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_k, 1.0, True, _Layout.packed, True, True)
    out, low = out.double().cpu(), low.view(out.shape).double().cpu()
    for n in range(len(lens_q)):
        for i in range(at_q[n], at_q[n + 1]):
            seen = v[at_k[n]:at_k[n + 1] - (at_q[n + 1] - 1 - i)].double().repeat_interleave(2, 1)
            if len(seen) == 0:
                continue
            sums = (len(seen) + 24) * 2.0 ** -24 * seen.abs().mean(0)
            step = _spacing(out[i], dtype) / 254
            assert low[i].abs().max() <= 127
            over = (out[i] + low[i] * step - seen.mean(0)).abs() - (0.5 + 2.0 ** -12) * step - sums
            assert over.max() <= 0, (i, over.max().item(), step.max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 136])
@pytest.mark.parametrize("lens_q,lens_k", _WRITERS)
def test_gradients_without_the_outputs_rounding(lens_q, lens_k, D, dtype):
    """Values that are half a and half the type's next value: their mean, the output, lies between the two and its
    rounding is as large as every dout . v - delta.  delta of the rounded output misses by |dout| times half a step, all
    of ds; delta as it is by a 254th of that, and the bound below is made of the latter."""
    from kernels.attention import forge_varlen_attention

    eps = torch.finfo(dtype).eps
    unit, tiny = _unit(dtype)
    T, Tk, u32 = sum(lens_q), sum(lens_k), 2.0 ** -24
    q = torch.full((T, 2, D), 2.0 ** -6, dtype=dtype)
    k = torch.ones(Tk, 1, D, dtype=dtype)
    v = torch.full((Tk, 1, D), 1.5, dtype=dtype)
    v[1::2] += eps
    do = (torch.rand(T, 2, D, generator=torch.Generator().manual_seed(0)) + 0.5).to(dtype)
    at_q, at_k = _offsets(lens_q), _offsets([n // 2 * 2 for n in lens_k])
    cu_q, cu_k = (torch.tensor(a, device="cuda", dtype=torch.int32) for a in (at_q, at_k))
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    out = forge_varlen_attention(*leaves, cu_q, cu_k, causal=False, scale=1.0)
    dq, dk = (t.double().cpu() for t in torch.autograd.grad(out, leaves[:2], do.cuda()))
    want_dk, err_dk = torch.zeros(Tk, D).double(), torch.zeros(Tk, D).double()
    for n in range(len(lens_q)):
        rows, keys = slice(at_q[n], at_q[n + 1]), slice(at_k[n], at_k[n + 1])
        m = at_k[n + 1] - at_k[n]
        for h in range(2):
            r = head_fwd_bwd(q[rows, h], k[keys, 0], v[keys, 0], do[rows, h], 1.0, False, 0.0, 0.0)
            d = do[rows, h].double()
            sums = (D + m + 24) * u32 * 1.6 * d.sum(-1)  # of dout . v, of delta, and of the output in it
            delta_err = (0.5 + 2.0 ** -12) / 254 * eps * d.sum(-1) + 2 * sums
            ds = (d @ v[keys, 0].double().T - (d * r.o).sum(-1, keepdim=True)) / m
            rel = (2 * D * 2.0 ** -6 * (D + 8) + 2 * m + 32) * u32  # of a probability
            ds_err = (delta_err.unsqueeze(1) + sums.unsqueeze(1)) / m + ds.abs() * (unit + 4 * rel) + tiny * 2.0 ** -14
            bound = (ds_err.sum(1) + (m + 16) * u32 * ds.abs().sum(1)).unsqueeze(1) * torch.ones(D) + tiny
            missed = 0.4 * eps * d.sum(-1, keepdim=True)  # (what delta of the rounded output would do to dq)
            assert bool((bound < 0.5 * missed).all())
            assert bool(((dq[rows, h] - r.dq).abs() <= bound).all()), (n, h)
            want_dk[keys] += r.dk
            err_dk[keys] += (ds_err + (len(d) + 16) * u32 * ds.abs()).T @ q[rows, h].double()
    assert bool(((dk[:, 0] - want_dk).abs() <= err_dk + want_dk.abs() * unit + tiny).all())


@pytest.mark.gpu
def test_a_cache_with_room_to_grow():
    """Tokens appended in place: sequences without queries stand for the room behind each sequence's keys, whatever it
    holds.  Steps of one and more tokens, eager and in a captured call that is replayed as the offsets move."""
    from kernels.attention import forge_varlen_attention

    H, kv, D, room, held = 8, 2, 64, [700, 40, 300], [600, 0, 129]
    starts, steps = _offsets(room), 6
    g = torch.Generator().manual_seed(0)
    cache = torch.full((2, sum(room) + 500, kv, D), float("nan"), dtype=BF16)
    for s, n in zip(starts, held):
        cache[:, s:s + n] = torch.randn(2, n, kv, D, generator=g).to(BF16)
    kc, vc = cache.cuda()
    q = torch.zeros(3, H, D, dtype=BF16, device="cuda")
    # a sequence of the batch, then its room, which has no queries
    cu_q = torch.tensor([0, 1, 1, 2, 2, 3, 3], dtype=torch.int32, device="cuda")
    cu_k = torch.zeros(7, dtype=torch.int32, device="cuda")

    def step():
        return forge_varlen_attention(q, kc, vc, cu_q, cu_k)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for t in range(steps):
        new = torch.randn(2, 3, kv, D, generator=g).to(BF16)
        for i, s in enumerate(starts[:3]):
            cache[:, s + held[i]] = new[:, i]
            kc[s + held[i]], vc[s + held[i]] = new[0, i].cuda(), new[1, i].cuda()
            held[i] += 1
        q.copy_(torch.randn(3, H, D, generator=g).to(BF16))
        cu_k.copy_(torch.tensor([x for i, s in enumerate(starts[:3]) for x in (s, s + held[i])] + [starts[3]], dtype=torch.int32))
        out = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, captured), t
        for i, s in enumerate(starts[:3]):
            keys = slice(s, s + held[i])
            for h in range(H):
                r = head_fwd_bwd(q[i:i + 1, h].cpu(), cache[0, keys, h * kv // H], cache[1, keys, h * kv // H],
                                 torch.zeros(1, D), D ** -0.5, True, *_unit(BF16))
                _within(out[i:i + 1, h], r.o, r.o_err, (t, i, h))


def test_scales_that_fp32_cannot_divide_by_are_refused():
    from forge_hip import _lib as L
    from kernels.attention import forge_varlen_attention

    t, cu = torch.zeros(4, 2, 64, dtype=BF16), torch.tensor([0, 4], dtype=torch.int32)
    rows = [16, 0, 512, 64]
    for scale in (1e-38, 1e-31, 1e31):
        with pytest.raises(ValueError, match="positive, from"):
            forge_varlen_attention(t, t, t, cu, scale=scale)
        assert L.forge_attention_fwd(2, *(rows * 4), None, None, 16, 16, 1, 4, 4, 4, 2, 64, scale, 1, None, None) == 1
        assert b"scale" in L.forge_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-20])
def test_small_scales(scale):
    _check([70, 3], [70, 40], 4, 2, 64, BF16, scale=scale)
