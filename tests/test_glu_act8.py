"""Gated activation kept in 8 bits for the backward pass (`glu_act8`).

What is kept is compared exactly (a power of two and an integer).  Other
tolerances, derived before the first run, with U = 2^-24 and x the kept value:
a result is rounded once (finfo.eps / 2 relative) after fp32 arithmetic, whose
error is
  silu: e^-x has a relative error of (1.5 |x| + 3) U from its argument and the
    exponential, which reaches s = 1 / (1 + e^-x) by a factor 1 - s; with the
    reciprocal and the product act is within k = ((1.5 |x| + 3) (1 - s) + 4) U
    of |act|, and the slope s (1 + x (1 - s)) within k of s (1 + |x|) plus U s
    |x| for 1 - s (exact past |x| = 100, where s is 1 or nearly 0); the
    reciprocal may give 0 for an s below 2^-126;
  tanh form: the exponent 2u, u = 0.8 x (1 + 0.045 x^2), has 5 roundings, so
    act is within (15 |u| + 8) U and the slope's terms within (30 |u| + 20) U;
  exact form: the polynomial's 1.5e-7 of erf and its evaluation's 2e-7 put the
    normal distribution function within 3e-7, act within 3e-7 |x| and the slope
    within 4e-7.
Products with dout and up add 3 roundings.
"""
import math

import pytest
import torch

from oracle.glu_act8 import GROUP, act_and_slope, fwd_bwd, kept

U = 2.0 ** -24
ACTS = ["silu", "gelu_tanh", "gelu_exact"]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _bounds(x, activation):
    """Error bounds of (act, slope) at x (float64)."""
    act, slope = act_and_slope(x, activation)
    a = x.abs()
    if activation == "silu":
        s, far = torch.sigmoid(x), a > 100
        k = torch.where(far, 4.0, (1.5 * a + 3) * (1 - s) + 4) * U
        flush = 2.0 ** -126 * (1 + a)
        return k * act.abs() + flush, torch.where(far, 4 * U * slope.abs(), (k * (1 + a) + U * a) * s) + flush
    if activation == "gelu_tanh":
        u = math.sqrt(2 / math.pi) * a * (1 + 0.044715 * a * a)
        es = torch.sigmoid(2 * u * x.sign())
        terms = es + 2 * a * es * (1 - es) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * a * a)
        # past 100 the slope is exactly that at 100
        return torch.where(a > 100, U, (15 * u + 8) * U) * act.abs(), torch.where(a > 100, U, (30 * u + 20) * U) * terms
    return 3e-7 * a + 2 * U * act.abs(), torch.full_like(a, 4e-7)


def _within(got, ref, err, what):
    eps, tiny = torch.finfo(got.dtype).eps, torch.finfo(got.dtype).smallest_normal
    got = got.double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), f"{what}: NaN in other places"
    # what leaves the type's range rounds to an infinity; denormals have a spacing of their own
    most = torch.finfo(torch.float32).max if eps < 1e-6 else (65504.0 if eps < 2e-3 else 3.3e38)
    ok = ref.abs() < most * 0.999
    bound = (ref.abs() + err) * (eps / 2) + err * (1 + eps) + tiny * eps
    off = ((got - ref).abs() - bound)[ok & ~ref.isnan()]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: off by {off.max():.3e} more than the bound"


def _check(gate, up, dout, activation, call):
    """call(gate, up) -> (out, dgate, dup) on the GPU, against the oracle."""
    out, dgate, dup = call(gate, up)
    cols = gate.shape[-1]
    g2, u2, d2 = (t.reshape(-1, cols).cpu() for t in (gate, up, dout))
    r_out, r_dg, r_du = fwd_bwd(g2, u2, d2, activation)
    x, u, d = kept(g2), kept(u2), d2.double()
    ea = _bounds(g2.double(), activation)[0]
    ka, ks = _bounds(x, activation)
    _within(out.reshape(-1, cols), r_out, ea * u2.double().abs() + 2 * U * r_out.abs(), "out")
    _within(dgate.reshape(-1, cols), r_dg, ks * (d * u).abs() + 3 * U * r_dg.abs(), "dgate")
    _within(dup.reshape(-1, cols), r_du, ka * d.abs() + 2 * U * r_du.abs(), "dup")


def _plain_call(dout, activation):
    from kernels.glu_act8 import glu_act8

    def call(gate, up):
        gate, up = gate.detach().requires_grad_(True), up.detach().requires_grad_(True)
        out = glu_act8(gate, up, activation)
        return (out.detach(), *torch.autograd.grad(out, (gate, up), dout))

    return call


def _decode(buf, rows, cols):
    """(gate, up) that a kept buffer stands for, from its documented layout."""
    pitch = -(-cols // GROUP) * GROUP
    buf = buf.cpu()
    q = buf[: 2 * rows * pitch].view(torch.int8).view(2, rows, -1, GROUP).double()
    e = buf[2 * rows * pitch:].view(rows, -1, 2).permute(2, 0, 1).unsqueeze(-1).to(torch.int32) - 127
    v = torch.where(q == -128, float("nan"), torch.ldexp(q, e)).reshape(2, rows, pitch)
    return v[0, :, :cols], v[1, :, :cols]


def _awkward(rows, cols, dtype, seed):
    """Groups of very different size, zeros, ties and largest values at the border of a scale."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    far = {torch.float32: 100, torch.bfloat16: 100, torch.float16: 10}[dtype]
    groups = -(-cols // GROUP)
    size = torch.randint(-far, far + 1, (rows, groups), generator=g).repeat_interleave(GROUP, 1)[:, :cols]
    x = torch.ldexp(x, size)
    kind = torch.randint(0, 5, (rows, groups), generator=g).repeat_interleave(GROUP, 1)[:, :cols]
    x = torch.where(kind == 0, 0.0, x)
    # integers and halves, whose largest may be 127 or 127.5: exact borders and ties
    halves = torch.randint(-255, 256, (rows, cols), generator=g) / 2
    x = torch.where(kind == 1, halves, x)
    return x.to(dtype)


# ---------------------------------------------------------------------------
# the oracle and the refusals (CPU)
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("activation", ACTS)
def test_oracle_slopes_against_differences(activation):
    x = torch.linspace(-6, 6, 41, dtype=torch.float64)
    h = 1e-6
    numeric = (act_and_slope(x + h, activation)[0] - act_and_slope(x - h, activation)[0]) / (2 * h)
    torch.testing.assert_close(act_and_slope(x, activation)[1], numeric, rtol=1e-7, atol=1e-8)


def test_oracle_kept_values():
    x = torch.zeros(1, 64, dtype=torch.float64)
    x[0, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])       # scale 1: halves go to even
    x[0, 32:36] = torch.tensor([127.5, 1.0, 3.0, -127.0])  # scale 2
    v = kept(x)[0]
    assert v[:4].tolist() == [127.0, 0.0, 2.0, -2.0]
    assert v[32:36].tolist() == [128.0, 0.0, 4.0, -128.0]
    x[0, 1], x[0, 33] = float("inf"), float("nan")
    v = kept(x)[0]
    assert v[0] == 127.0 and v[1].isnan() and v[33].isnan() and v[32] == 128.0
    g = torch.Generator().manual_seed(0)
    y = torch.randn(8, 320, generator=g, dtype=torch.float64)
    assert ((kept(y) - y).abs().view(8, 10, 32) <= y.view(8, 10, 32).abs().amax(-1, keepdim=True) / 127).all()


def test_refusals():
    from kernels.glu_act8 import glu_act8, glu_act8_packed

    a = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="same shape"):
        glu_act8(a, a[:, :4])
    with pytest.raises(TypeError, match="same dtype"):
        glu_act8(a, a.half())
    with pytest.raises(TypeError, match="fp16, bf16, and fp32"):
        glu_act8(a.double(), a.double())
    with pytest.raises(ValueError, match="activation must be one of"):
        glu_act8(a, a, "relu")
    with pytest.raises(ValueError, match="must be even"):
        glu_act8_packed(torch.zeros(2, 7))
    with pytest.raises(TypeError, match="fp16, bf16, and fp32"):
        glu_act8_packed(a.long())
    for call in (lambda: glu_act8(a, a), lambda: glu_act8_packed(a)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def test_c_entry_errors():
    from forge_hip import _lib as L

    assert L.forge_glu_act8_bytes(3, 33) == 2 * 3 * 64 + 2 * 3 * 2 and L.forge_glu_act8_bytes(0, 5) == 0
    fwd = L.forge_glu_act8_fwd
    assert fwd(2, 3, 16, 8, 16, 8, 16, 8, 16, 2, 8, None) == 1 and b"activation 3" in L.forge_last_error()
    assert fwd(3, 0, 16, 8, 16, 8, 16, 8, 16, 2, 8, None) == 2
    assert fwd(2, 0, 16, 7, 16, 8, 16, 8, 16, 2, 8, None) == 1 and b"leading dimension" in L.forge_last_error()
    assert fwd(2, 0, 16, 8, 16, 8, 16, 8, 8, 2, 8, None) == 1 and b"misaligned" in L.forge_last_error()
    assert fwd(2, 0, 17, 8, 16, 8, 16, 8, 16, 2, 8, None) == 1
    assert fwd(2, 0, 16, 1 << 20, 16, 1 << 20, 16, 1 << 20, 16, 1 << 20, 1 << 20, None) == 2
    assert fwd(2, 0, 16, 8, 16, 8, 16, 8, 16, -1, 8, None) == 1
    assert fwd(2, 0, None, 0, None, 0, None, 0, None, 0, 8, None) == 0
    assert L.forge_glu_act8_bwd(2, 0, 16, 8, None, 16, 16, 8, 2, 8, None) == 1 and b"kept" in L.forge_last_error()


# ---------------------------------------------------------------------------
# the kernels
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 15), (3, 16), (2, 17), (5, 31), (4, 32), (7, 33), (2, 100),
                                       (3, 4097), (130, 1000)])
def test_shapes(rows, cols, dtype, activation):
    g = torch.Generator().manual_seed(rows * 7919 + cols)
    gate, up, dout = (torch.randn(rows, cols, generator=g).mul_(2.0).to(dtype).cuda() for _ in range(3))
    _check(gate, up, dout, activation, _plain_call(dout, activation))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("cols", [64, 333])
def test_kept_values_are_exact(cols, dtype):
    from kernels.glu_act8 import glu_act8

    rows = 200
    gate, up = _awkward(rows, cols, dtype, 1), _awkward(rows, cols, dtype, 2)
    gate[3, 5], gate[3, 40], up[4, 7] = float("inf"), float("nan"), float("-inf")
    if dtype == torch.float32:
        gate[6, :32] = torch.linspace(-1, 1, 32) * 1e-40   # below the least scale's half step: zeros
        gate[7, :32] = torch.linspace(-1, 1, 32) * 3e38
    out = glu_act8(gate.cuda().requires_grad_(True), up.cuda().requires_grad_(True))
    (buf,) = out.grad_fn.saved_tensors
    got = _decode(buf, rows, cols)
    for v, x in zip(got, (gate, up)):
        torch.testing.assert_close(v, kept(x), rtol=0, atol=0, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_large_small_and_non_finite_values(dtype, activation):
    gate, up = _awkward(64, 96, dtype, 5), _awkward(64, 96, dtype, 6).clamp(-8, 8)
    gate[1, 3], up[2, 4] = float("nan"), float("nan")
    g = torch.Generator().manual_seed(0)
    dout = torch.randn(64, 96, generator=g).to(dtype).cuda()
    # an infinite gate's own output follows the formula; its kept value is NaN
    _check(gate.cuda(), up.cuda(), dout, activation, _plain_call(dout, activation))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_strides(dtype):
    """Rows of a wider buffer that begin off 16 bytes, a batch of 3-D slices,
    expanded rows, a transposed tensor, and an expanded gradient."""
    from kernels.glu_act8 import glu_act8

    g = torch.Generator().manual_seed(9)
    wide = torch.randn(2, 7, 103, generator=g).to(dtype).cuda()
    dense = torch.randn(2, 7, 50, generator=g).to(dtype).cuda()
    dout = torch.randn(2, 7, 50, generator=g).to(dtype).cuda()
    pairs = [(wide[..., 1:51], wide[..., 53:]),
             (dense[:, :1].expand(2, 7, 50), dense),
             (torch.randn(2, 50, 7, generator=g).to(dtype).cuda().transpose(1, 2), wide[..., 2:52])]
    for gate, up in pairs:
        _check(gate, up, dout, "silu", _plain_call(dout, "silu"))
    one = torch.ones(1, 1, 1, device="cuda", dtype=dtype).expand(2, 7, 50)
    _check(dense, dense, one, "gelu_tanh", _plain_call(one, "gelu_tanh"))
    column = torch.randn(5, 3, generator=g).to(dtype).cuda()[:, 1:2]
    d1 = torch.ones(5, 1, device="cuda", dtype=dtype)
    _check(column, column, d1, "silu", _plain_call(d1, "silu"))
    with torch.no_grad():
        a = glu_act8(wide[..., 1:51], wide[..., 53:])
    b = glu_act8(wide[..., 1:51].detach().requires_grad_(True), wide[..., 53:])
    assert torch.equal(a, b) and b.grad_fn is not None and not a.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("cols", [5, 64, 4097])
def test_packed_equals_separate(cols, activation):
    from kernels.glu_act8 import glu_act8, glu_act8_packed

    g = torch.Generator().manual_seed(cols)
    gate_up = torch.randn(3, 11, 2 * cols, generator=g).to(torch.bfloat16).cuda().requires_grad_(True)
    dout = torch.randn(3, 11, cols, generator=g).to(torch.bfloat16).cuda()
    gate, up = (t.detach().requires_grad_(True) for t in gate_up.chunk(2, -1))
    a, b = glu_act8_packed(gate_up, activation), glu_act8(gate, up, activation)
    assert torch.equal(a, b)
    (da,) = torch.autograd.grad(a, gate_up, dout)
    assert torch.equal(da, torch.cat(torch.autograd.grad(b, (gate, up), dout), -1))
    with torch.no_grad():
        assert torch.equal(glu_act8_packed(gate_up, activation), a)


@pytest.mark.gpu
def test_inputs_are_untouched_and_freed_and_empty_calls():
    from kernels.glu_act8 import glu_act8, glu_act8_packed

    x = torch.randn(512, 4096, device="cuda", dtype=torch.bfloat16)
    gate, up = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    base = torch.cuda.memory_allocated()
    out = glu_act8(gate * 1.0, up * 1.0)  # projections' outputs: nothing else holds them
    held = torch.cuda.memory_allocated() - base
    n = x.numel()
    assert held <= 2 * n + 2 * n + n // 16 + 4096  # out, the 8-bit copy and its scales
    out.backward(torch.ones_like(out))
    assert torch.equal(gate, x) and torch.equal(up, x)
    for shape in ((0, 32), (3, 0)):
        e = torch.zeros(shape, device="cuda", requires_grad=True)
        o = glu_act8(e, e)
        assert o.shape == shape and torch.autograd.grad(o.sum(), e)[0].shape == shape
    p = torch.zeros(2, 0, device="cuda", requires_grad=True)
    assert glu_act8_packed(p).shape == (2, 0)


@pytest.mark.gpu
def test_shared_input_and_second_backward():
    """gate and up the same tensor (gradients add up), the same graph walked twice."""
    from kernels.glu_act8 import glu_act8

    g = torch.Generator().manual_seed(3)
    x = torch.randn(9, 70, generator=g).cuda().requires_grad_(True)
    dout = torch.randn(9, 70, generator=g).cuda()
    out = glu_act8(x, x)
    (a,) = torch.autograd.grad(out, x, dout, retain_graph=True)
    (b,) = torch.autograd.grad(out, x, dout)
    assert torch.equal(a, b)
    _, dg, du = fwd_bwd(x.detach().cpu(), x.detach().cpu(), dout.cpu(), "silu")
    torch.testing.assert_close(a.double().cpu(), dg + du, rtol=64 * U, atol=64 * U * float((dg.abs() + du.abs()).max()))


@pytest.mark.gpu
def test_side_stream_and_graph():
    from kernels.glu_act8 import glu_act8

    gate, up, dout = (torch.randn(33, 500, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    leaves = [gate.clone().requires_grad_(True), up.clone().requires_grad_(True)]

    def step(args):
        out = glu_act8(*args, "gelu_tanh")
        return (out, *torch.autograd.grad(out, args, dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(leaves)
    fresh = [t.detach().clone().requires_grad_(True) for t in leaves]
    for i in range(4):
        for a, b in zip(leaves, fresh):
            b.detach().normal_()
            a.detach().copy_(b)
        dout.normal_()
        graph.replay()
        eager = step(fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager)), i


@pytest.mark.gpu
def test_more_than_2_31_values():
    """Offsets past 32 bits in every buffer, checked on the last rows."""
    from kernels.glu_act8 import glu_act8

    rows, cols = (1 << 31) // 16384 + 3, 16384
    x = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    last = torch.randn(3, cols, generator=g).to(torch.bfloat16).cuda()
    x[-3:] = last
    x.requires_grad_(True)
    out = glu_act8(x, x.detach())
    (dx,) = torch.autograd.grad(out, x, torch.ones(1, 1, device="cuda", dtype=torch.bfloat16).expand(rows, cols))
    small = last.clone().requires_grad_(True)
    want = glu_act8(small, last)
    (dw,) = torch.autograd.grad(want, small, torch.ones_like(want))
    assert torch.equal(out[-3:], want) and torch.equal(dx[-3:], dw) and out[:-3].abs().sum() == 0
