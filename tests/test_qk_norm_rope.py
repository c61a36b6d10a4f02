"""RMS norm of q and k heads + RoPE in one pass (`apply_qk_norm_rope`).

Tolerances, derived before the first run: an output is rounded once, by at
most half a step of its type (finfo.eps / 2 relative), after fp32 arithmetic.
The longest chain of an output is the sum of squares (at most 16 products in a
lane, 6 shuffles), rsqrt, and 6 products and sums: fewer than 32 roundings of
2^-24 relative to the terms that are added, which the oracle returns.  A
gradient adds the second sum over the head: fewer than 64.  A weight gradient
adds at most rows-per-lane + 12 terms on top; the sizes here stay below 128.
"""
import pytest
import torch

from oracle.qk_norm_rope import forward as oracle_forward
from oracle.qk_norm_rope import head_fwd_bwd

U = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _cos_sin(rows, dim, dtype):
    inv = 1.0 / 10000.0 ** (torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    ang = torch.arange(rows, dtype=torch.float64).unsqueeze(1) * inv
    ang = torch.cat([ang, ang], 1)
    return ang.cos().to(dtype).unsqueeze(0), ang.sin().to(dtype).unsqueeze(0)


def _make(b, nq, nk, s, d, dtype, layout="bshd", seed=0, device="cuda"):
    """q, k in one of the layouts that callers pass."""
    g = torch.Generator().manual_seed(seed)
    if layout == "packed":  # columns of one projection's output
        qkv = torch.randn(b, s, nq + 2 * nk, d, generator=g).to(dtype).to(device)
        return qkv[:, :, :nq].transpose(1, 2), qkv[:, :, nq:nq + nk].transpose(1, 2)
    out = []
    for n in (nq, nk):
        if layout == "bhsd":
            out.append(torch.randn(b, n, s, d, generator=g).to(dtype).to(device))
        elif layout == "bshd":
            out.append(torch.randn(b, s, n, d, generator=g).to(dtype).to(device).transpose(1, 2))
        else:  # "odd": rows that begin off a 16-byte boundary
            t = torch.randn(b * n * s * d + 1, generator=g).to(dtype).to(device)
            out.append(t[1:].view(b, n, s, d))
    return tuple(out)


def _within(got, ref, terms, k, what):
    eps = torch.finfo(got.dtype).eps
    # half a step of the stored type, k fp32 roundings of the terms, and the spacing of fp16's subnormals
    bound = ref.abs() * (eps / 2) + terms * (k * U * (1 + eps)) + torch.finfo(got.dtype).smallest_normal * eps
    err = (got.double().cpu() - ref).abs()
    worst = (err - bound).max().item() if err.numel() else -1.0
    assert worst <= 0, f"{what}: off by {worst:.3e} more than the bound"


def _run(q, k, qw, kw, cos, sin, positions, offset, eps=1e-6, seed=1, train_weights=True, dense_grads=True):
    from kernels.rope import apply_qk_norm_rope

    g = torch.Generator().manual_seed(seed)
    q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    qw, kw = (w.detach().requires_grad_(train_weights) for w in (qw, kw))
    oq, ok = apply_qk_norm_rope(q, k, qw, kw, cos, sin, positions=positions, eps=eps, offset=offset)
    assert oq.shape == q.shape and ok.shape == k.shape and oq.dtype == q.dtype
    dq = torch.randn(q.shape, generator=g).to(q.dtype).cuda()
    dk = torch.randn(k.shape, generator=g).to(k.dtype).cuda()
    if not dense_grads:
        dq, dk = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (dq, dk))
    leaves = [q, k] + ([qw, kw] if train_weights else [])
    grads = torch.autograd.grad((oq, ok), leaves, (dq, dk))
    return (oq, ok), grads, (dq, dk)


def _check(q, k, qw, kw, cos, sin, positions, offset, eps=1e-6, **kw_run):
    outs, grads, dos = _run(q, k, qw, kw, cos, sin, positions, offset, eps, **kw_run)
    b, _, s, d = q.shape
    c, sn = cos.cpu(), sin.cpu()
    if positions is not None:
        p = positions.cpu().view(b, s)
        batch = torch.arange(b).view(b, 1) if c.shape[0] == b else torch.zeros(1, 1, dtype=torch.long)
        c, sn = c[batch, p], sn[batch, p]
    for i, (x, w, do) in enumerate(((q, qw, dos[0]), (k, kw, dos[1]))):
        ref = head_fwd_bwd(x.cpu(), w.cpu(), c, sn, do.cpu(), eps, offset)
        _within(outs[i], ref.out, ref.out_terms, 32, f"out[{i}]")
        _within(grads[i], ref.dx, ref.dx_terms, 64, f"dx[{i}]")
        if len(grads) == 4:
            _within(grads[2 + i], ref.dw, ref.dw_terms, 128, f"dw[{i}]")


def _weights(d, dtype, offset, device="cuda", seed=3):
    g = torch.Generator().manual_seed(seed)
    return tuple((torch.randn(d, generator=g) * 0.2 + 1.0 - offset).to(dtype).to(device) for _ in range(2))


# ---------------------------------------------------------------------------
# the oracle and the refusals (CPU)
# ---------------------------------------------------------------------------
def test_oracle_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, 4, 6, generator=g, dtype=torch.float64, requires_grad=True)
    w = (1 + 0.2 * torch.randn(6, generator=g, dtype=torch.float64)).requires_grad_(True)
    cos, sin = _cos_sin(4, 6, torch.float64)
    c, s = cos[..., :3].unsqueeze(1), sin[..., :3].unsqueeze(1)
    assert torch.autograd.gradcheck(lambda a, b: oracle_forward(a, b, c, s, 1e-6, 0.5), (x, w))
    do = torch.randn(2, 3, 4, 6, generator=g, dtype=torch.float64)
    ref = head_fwd_bwd(x.detach(), w.detach(), cos, sin, do, 1e-6, 0.5)
    out = oracle_forward(x, w, c, s, 1e-6, 0.5)
    dx, dw = torch.autograd.grad(out, (x, w), do)
    torch.testing.assert_close(ref.out, out.detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(ref.dx, dx, rtol=1e-10, atol=1e-12)
    torch.testing.assert_close(ref.dw, dw, rtol=1e-10, atol=1e-12)
    for value, terms in ((ref.out, ref.out_terms), (ref.dx, ref.dx_terms), (ref.dw, ref.dw_terms)):
        assert (value.abs() <= terms * (1 + 1e-9) + 1e-12).all()


def test_refusals():
    from kernels.rope import apply_qk_norm_rope

    q, k = _make(2, 4, 2, 5, 8, FP32, device="cpu")
    qw, kw = _weights(8, FP32, 0.0, "cpu")
    cos, sin = _cos_sin(5, 8, FP32)

    def bad(error, match, **change):
        a = {"q": q, "k": k, "q_weight": qw, "k_weight": kw, "cos": cos, "sin": sin, **change}
        with pytest.raises(error, match=match):
            apply_qk_norm_rope(**a)

    bad(ValueError, "batch, heads, seq, head_dim", q=q[0])
    bad(ValueError, "does not match", k=k[:, :, :4])
    bad(ValueError, "does not match", k=k[:1])
    odd = torch.zeros(2, 4, 5, 7)
    bad(ValueError, "head_dim must be even", q=odd, k=odd)
    wide = torch.zeros(1, 1, 1, 1026)
    bad(ValueError, "at most 1024", q=wide, k=wide)
    bad(TypeError, "fp16, bf16 or fp32", q=q.double(), k=k.double())
    bad(TypeError, "same dtype", k=k.to(BF16))
    bad(ValueError, r"must be \[8\]", q_weight=qw[:4])
    bad(TypeError, "same dtype", k_weight=kw.to(BF16))
    bad(ValueError, "cos and sin", sin=sin[:, :4])
    bad(ValueError, "cos and sin", cos=cos.expand(3, 5, 8), sin=sin.expand(3, 5, 8))
    bad(ValueError, "5 rows", q=q[:, :, :3], k=k[:, :, :3])
    bad(TypeError, "floating point", cos=cos.long(), sin=sin.long())
    bad(TypeError, "integer tensor", positions=torch.zeros(2, 5))
    bad(ValueError, "10 entries", positions=torch.zeros(2, 4, dtype=torch.long))
    bad(ValueError, "eps", eps=-1.0)
    bad(RuntimeError, "ROCm GPU")  # a CPU call that is otherwise right


def test_c_entry_errors():
    from forge_hip import _lib as L

    s4, table = [16, 0, 0, 0], [16, 0, 0, 16, 0, 0]

    def fwd(dtype=2, w=2, t=2, rows=8, sizes=(1, 4, 2, 8, 128)):
        return L.forge_qk_norm_rope_fwd(dtype, *s4 * 4, 16, 16, w, *table, t, rows, None, *sizes, 1e-6, 0.0, None)

    assert fwd(sizes=(1, 4, 2, 8, 127)) == 1 and b"head_dim 127" in L.forge_last_error()
    assert fwd(sizes=(1, 4, 2, 8, 2048)) == 1
    assert fwd(sizes=(1, -4, 2, 8, 128)) == 1 and b"negative" in L.forge_last_error()
    assert fwd(dtype=3) == 2 and fwd(w=3) == 2
    assert fwd(t=1) == 2 and b"cos/sin dtype" in L.forge_last_error()
    assert fwd(rows=7) == 1 and b"7 rows" in L.forge_last_error()
    assert fwd(sizes=(1 << 20, 4096, 2, 1, 128)) == 2 and b"2^30" in L.forge_last_error()
    assert fwd(sizes=(0, 4, 2, 8, 128)) == 0
    rc = L.forge_qk_norm_rope_bwd(2, *s4 * 6, 16, 16, 2, *table, 2, 8, None, 16, None, None, 1, 4, 2, 8, 128, 1e-6, 0.0,
                                  None)
    assert rc == 1 and b"workspace" in L.forge_last_error()


# ---------------------------------------------------------------------------
# the kernels
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("d", [2, 6, 32, 64, 80, 96, 128, 256, 510, 512, 1024])
def test_head_dims(d, dtype):
    q, k = _make(2, 5, 3, 9, d, dtype)
    cos, sin = (t.cuda() for t in _cos_sin(9, d, dtype))
    _check(q, k, *_weights(d, dtype, 0.0), cos, sin, None, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["bhsd", "bshd", "packed", "odd"])
@pytest.mark.parametrize("b,nq,nk,s,d", [(1, 1, 1, 1, 128), (3, 7, 2, 1, 64), (1, 32, 8, 77, 128), (2, 4, 4, 300, 96)])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
def test_layouts(layout, b, nq, nk, s, d, dtype):
    q, k = _make(b, nq, nk, s, d, dtype, layout)
    cos, sin = (t.cuda() for t in _cos_sin(s, d, dtype))
    _check(q, k, *_weights(d, FP32, 1.0), cos, sin, None, 1.0, dense_grads=layout != "bhsd")


@pytest.mark.gpu
@pytest.mark.parametrize("wdtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("d", [64, 72, 128, 256])
def test_weights_of_another_type(d, dtype, wdtype):
    for layout in ("bshd", "bhsd"):
        q, k = _make(2, 5, 3, 9, d, dtype, layout)
        cos, sin = (t.cuda() for t in _cos_sin(9, d, dtype))
        _check(q, k, *_weights(d, wdtype, 0.0), cos, sin, None, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("wdtype", [BF16, FP16], ids=str)
def test_narrow_weights_of_many_tokens(wdtype):
    q, k = _make(2, 32, 8, 1100, 128, FP32)  # more workgroups than ask for the weights late
    cos, sin = (t.cuda() for t in _cos_sin(1100, 128, FP32))
    _check(q, k, *_weights(128, wdtype, 1.0), cos, sin, None, 1.0, train_weights=False)


@pytest.mark.gpu
@pytest.mark.parametrize("batched", [False, True])
@pytest.mark.parametrize("tdtype", [BF16, FP32], ids=str)
def test_positions_and_tables(batched, tdtype):
    b, s, d, rows = 3, 21, 128, 50
    q, k = _make(b, 8, 2, s, d, BF16)
    cos, sin = _cos_sin(rows, d, tdtype)
    if batched:  # another table for each batch row
        cos, sin = (torch.cat([t, t.flip(1), t.roll(3, 1)]) for t in (cos, sin))
    g = torch.Generator().manual_seed(5)
    pos = torch.randint(0, rows, (b, s), generator=g, dtype=torch.int32).cuda()
    _check(q, k, *_weights(d, BF16, 0.0), cos.cuda(), sin.cuda(), pos, 0.0)


@pytest.mark.gpu
def test_positions_outside_the_table():
    from kernels.rope import apply_qk_norm_rope

    q, k = _make(1, 4, 2, 6, 64, BF16)
    qw, kw = _weights(64, BF16, 0.0)
    cos, sin = (t.cuda() for t in _cos_sin(8, 64, BF16))
    good = torch.tensor([0, 1, 2, 3, 4, 7], device="cuda")
    bad = torch.tensor([0, -1, 2, 8, 4, 1 << 40], device="cuda")
    a, b = apply_qk_norm_rope(q, k, qw, kw, cos, sin, good), apply_qk_norm_rope(q, k, qw, kw, cos, sin, bad)
    for x, y in zip(a, b):
        assert torch.equal(x[:, :, [0, 2, 4]], y[:, :, [0, 2, 4]])
        assert y[:, :, [1, 3, 5]].isnan().all() and not x.isnan().any()
    with pytest.raises(IndexError):
        apply_qk_norm_rope(q, k, qw, kw, cos, sin, bad, validate_positions=True)
    apply_qk_norm_rope(q, k, qw, kw, cos, sin, good, validate_positions=True)


@pytest.mark.gpu
def test_zero_rows_large_values_and_no_tokens():
    from kernels.rope import apply_qk_norm_rope

    q, k = _make(1, 2, 2, 4, 64, FP32)
    q = q.clone()
    q[0, 0, 1] = 0.0
    q[0, 1, 2] *= 1e15   # squares near 1e30
    k = k * 1e-12        # eps outweighs the squares
    cos, sin = (t.cuda() for t in _cos_sin(4, 64, FP32))
    _check(q, k, *_weights(64, FP32, 0.0), cos, sin, None, 0.0)
    empty = torch.zeros(2, 4, 0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    out = apply_qk_norm_rope(empty, empty[:, :1], w, w.detach(), cos[:, :0], sin[:, :0])
    assert out[0].shape == empty.shape
    dx, dw = torch.autograd.grad(out[0].sum() + out[1].sum(), (empty, w))
    assert dx.shape == empty.shape and torch.equal(dw, torch.zeros_like(dw))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
def test_no_eps_with_odd_heads(dtype):
    """eps = 0: nothing but the heads themselves may be divided by their norm."""
    q, k = _make(2, 5, 3, 7, 96, dtype)
    cos, sin = (t.cuda() for t in _cos_sin(7, 96, dtype))
    _check(q, k, *_weights(96, dtype, 0.0), cos, sin, None, 0.0, eps=0.0)


@pytest.mark.gpu
def test_a_head_with_an_infinity_or_nan_stays_alone():
    from kernels.rope import apply_qk_norm_rope

    q, k = _make(1, 4, 1, 3, 128, BF16)
    qw, kw = _weights(128, BF16, 0.0)
    cos, sin = (t.cuda() for t in _cos_sin(3, 128, BF16))
    clean = apply_qk_norm_rope(q, k, qw, kw, cos, sin)[0]
    q = q.clone()
    q[0, 1, 1, 5], q[0, 2, 0, 70] = float("inf"), float("nan")
    got = apply_qk_norm_rope(q, k, qw, kw, cos, sin)[0]
    assert got[0, 1, 1].isnan().any() and got[0, 2, 0].isnan().all()
    touched = torch.zeros(4, 3, dtype=torch.bool)
    touched[1, 1] = touched[2, 0] = True
    assert torch.equal(got[0][~touched], clean[0][~touched])


@pytest.mark.gpu
def test_which_gradients_and_repeatable_sums():
    from kernels.rope import apply_qk_norm_rope

    q, k = _make(2, 32, 8, 257, 128, BF16)
    cos, sin = (t.cuda() for t in _cos_sin(257, 128, BF16))
    qw, kw = _weights(128, BF16, 0.0)
    _, frozen, _ = _run(q, k, qw, kw, cos, sin, None, 0.0, train_weights=False)
    _, first, _ = _run(q, k, qw, kw, cos, sin, None, 0.0)
    _, second, _ = _run(q, k, qw, kw, cos, sin, None, 0.0)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    assert torch.equal(frozen[0], first[0]) and torch.equal(frozen[1], first[1])
    # one weight alone; one output alone
    qr, kwr = q.detach().requires_grad_(True), kw.detach().requires_grad_(True)
    oq, ok = apply_qk_norm_rope(qr, k, qw, kwr, cos, sin)
    (only,) = torch.autograd.grad(ok, kwr, torch.ones_like(ok), retain_graph=True)
    dq, none = torch.autograd.grad(oq, (qr, kwr), torch.ones_like(oq))
    assert only.abs().sum() > 0 and none.abs().sum() == 0 and dq.shape == q.shape
    # under no_grad, the same values
    with torch.no_grad():
        again = apply_qk_norm_rope(qr, k, qw, kwr, cos, sin)
    assert torch.equal(again[0], oq) and torch.equal(again[1], ok) and not again[0].requires_grad


@pytest.mark.gpu
def test_expanded_heads_and_shared_weight():
    """k expanded over its heads (stride 0) and one weight for both norms: the
    gradients of what is shared add up."""
    from kernels.rope import apply_qk_norm_rope

    g = torch.Generator().manual_seed(2)
    d, s = 64, 5
    q = torch.randn(1, 4, s, d, generator=g).cuda().requires_grad_(True)
    k1 = torch.randn(1, 1, s, d, generator=g).cuda().requires_grad_(True)
    w = _weights(d, FP32, 0.0)[0].requires_grad_(True)
    cos, sin = (t.cuda() for t in _cos_sin(s, d, FP32))
    oq, ok = apply_qk_norm_rope(q, k1.expand(1, 3, s, d), w, w, cos, sin)
    do = torch.randn(1, 4, s, d, generator=g), torch.randn(1, 3, s, d, generator=g)
    dq, dk, dw = torch.autograd.grad((oq, ok), (q, k1, w), tuple(t.cuda() for t in do))
    rq = head_fwd_bwd(q.detach().cpu(), w.detach().cpu(), cos.cpu(), sin.cpu(), do[0], 1e-6, 0.0)
    rk = head_fwd_bwd(k1.detach().cpu().expand(1, 3, s, d), w.detach().cpu(), cos.cpu(), sin.cpu(), do[1], 1e-6, 0.0)
    _within(dq, rq.dx, rq.dx_terms, 64, "dq")
    _within(dk, rk.dx.sum(1, keepdim=True), rk.dx_terms.sum(1, keepdim=True), 68, "dk")
    _within(dw, rq.dw + rk.dw, rq.dw_terms + rk.dw_terms, 130, "dw")


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows of q more than 2^31 elements apart."""
    from kernels.rope import apply_qk_norm_rope

    d = 128
    far = (1 << 31) + 64
    buf = torch.zeros(far + 2 * d, device="cuda", dtype=BF16)
    g = torch.Generator().manual_seed(0)
    rows = torch.randn(2, 1, 1, d, generator=g).to(BF16).cuda()
    q = buf.as_strided((2, 1, 1, d), (far, d, d, 1))
    q.copy_(rows)
    cos, sin = (t.cuda() for t in _cos_sin(1, d, BF16))
    w = _weights(d, BF16, 0.0)
    got = apply_qk_norm_rope(q, rows, *w, cos, sin)
    want = apply_qk_norm_rope(rows, rows, w[0], w[1], cos, sin)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_side_stream_and_graph():
    """A decode step captured with a positions buffer that moves on, and the
    backward captured with leaves of its own; every replay against eager."""
    from kernels.rope import apply_qk_norm_rope

    q, k = _make(8, 32, 8, 1, 128, BF16)
    w = _weights(128, BF16, 0.0)
    cos, sin = (t.cuda() for t in _cos_sin(64, 128, BF16))
    pos = torch.zeros(8, 1, dtype=torch.long, device="cuda")
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, *w)]
    dq, dk = torch.randn_like(q), torch.randn_like(k)

    def step(args):
        with torch.no_grad():
            out = apply_qk_norm_rope(q, k, *w, cos, sin, pos)
        o = apply_qk_norm_rope(*args, cos, sin, pos)
        return (*out, *torch.autograd.grad(o, args, (dq, dk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(leaves)
    fresh = [t.detach().clone().requires_grad_(True) for t in (q, k, *w)]
    for i in range(4):
        pos.fill_(7 * i)
        q.normal_()
        for a, b in zip(leaves + fresh, (q, k, *w, q, k, *w)):
            a.detach().copy_(b)
        graph.replay()
        eager = step(fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager)), i
