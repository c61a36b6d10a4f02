"""RMS norm with the residual's addition (`add_rmsnorm`, `add_rmsnorm_int8`).

Tolerances, derived before the first run: a result is rounded once (half a step of
its type) after fp32 arithmetic.  The sum of squares adds at most 8 vectors of 8 in a
thread (rows of up to 16384 16-bit values; wider ones are read by more rounds, of
which the tests have at most 4), 6 shuffles and 4 waves: at most 330 roundings of
2^-24 in wide rows and 80 otherwise, of which rsqrt keeps half; 6 more follow.  A
gradient adds the second sum.  A weight gradient adds up to rows / workgroups + 80.
The 8-bit integers are those of exact arithmetic: equal."""
import pytest
import torch

from oracle.add_rmsnorm import fwd_bwd
from oracle.int8 import quantize

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _within(got, ref, terms, k, what):
    f = torch.finfo(got.dtype)
    bound = ref.abs() * (f.eps / 2) + terms * (k * U * (1 + f.eps)) + f.smallest_normal * f.eps
    over = (got.detach().double().cpu() - ref).abs() - bound
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, f"{what}: off by {worst:.3e} more than the bound"


def _make(rows, H, dtype, w_dtype, offset, seed=0, pad=0):
    """pad: columns between the rows of x and the residual (a slice of a wider buffer)."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, H + pad, generator=g).to(dtype)[:, :H]
    res = (torch.randn(rows, H + pad, generator=g) * 3).to(dtype)[:, :H]
    w = (torch.randn(H, generator=g) * 0.2 + 1.0 - offset).to(w_dtype)
    return x, res, w, torch.randn(rows, H, generator=g).to(dtype), torch.randn(rows, H, generator=g).to(dtype)


def _gpu(t):
    base = t._base if t._base is not None else t
    return torch.as_strided(base.cuda(), t.shape, t.stride(), t.storage_offset())


def _check(rows, H, dtype, w_dtype, offset=0.0, eps=1e-6, residual=True, stream_grad=True, **kw):
    from kernels.rmsnorm import add_rmsnorm

    x, res, w, dy, dh = _make(rows, H, dtype, w_dtype, offset, **kw)
    ref = fwd_bwd(x, res if residual else None, w, dy, dh if stream_grad else None, eps, offset)
    xg, wg = _gpu(x).requires_grad_(True), w.cuda().requires_grad_(True)
    rg = _gpu(res).requires_grad_(True) if residual else None
    y, h = add_rmsnorm(xg, rg, wg, eps=eps, offset=offset)
    assert torch.equal(h.detach().cpu(), ref.h), "h"
    k = 400 if H > 4096 else 100
    _within(y, ref.y, ref.y.abs(), k, "y")
    leaves = [t for t in (xg, rg, wg) if t is not None]
    outs, grads = ((y, h), (dy.cuda(), dh.cuda())) if stream_grad else ((y,), (dy.cuda(),))
    got = torch.autograd.grad(outs, leaves, grads)
    for t in got[:-1]:
        # (without a residual autograd adds the two parts, each rounded)
        extra = 0.0 if residual or not stream_grad else (ref.d_terms * torch.finfo(dtype).eps).max().item()
        _within(t, ref.d, ref.d_terms + extra / (2 * k * U), 2 * k, "d")
    _within(got[-1], ref.dw, ref.dw_terms, rows / min(rows, 512) + 180, "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,w_dtype", [(BF16, BF16), (FP16, FP32), (FP32, FP32), (FP32, BF16), (BF16, FP16)])
@pytest.mark.parametrize("rows,H", [(1, 1), (5, 7), (3, 64), (9, 511), (70, 1000), (6, 2048), (2, 2305), (33, 4096)])
def test_sizes_and_types(rows, H, dtype, w_dtype):
    _check(rows, H, dtype, w_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("H,dtype", [(8192, BF16), (8200, BF16), (16384, FP16), (16392, BF16), (20001, FP32), (9001, FP32)])
def test_wide_rows(H, dtype):
    _check(3, H, dtype, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [513, 2100, 9000])
def test_more_rows_than_workgroups(rows):
    _check(rows, 72, BF16, BF16)
    _check(min(rows, 2100), 1056, FP16, FP32)


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 8, 129])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rows_of_a_wider_buffer(dtype, pad):
    _check(11, 520, dtype, dtype, pad=pad)
    _check(11, 2056, dtype, dtype, pad=pad)


@pytest.mark.gpu
@pytest.mark.parametrize("residual,stream_grad", [(True, False), (False, True), (False, False)])
def test_without_a_residual_or_its_gradient(residual, stream_grad):
    _check(20, 1024, BF16, BF16, residual=residual, stream_grad=stream_grad)
    _check(20, 1003, FP32, FP32, offset=1.0, residual=residual, stream_grad=stream_grad)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [0.0, 1e-6, 1.0])
def test_offsets_and_eps(eps):
    _check(9, 333, BF16, BF16, offset=1.0, eps=eps)
    _check(9, 2560, FP32, FP32, offset=1.0, eps=eps)


@pytest.mark.gpu
def test_the_stream_alone_and_frozen_inputs():
    from kernels.rmsnorm import add_rmsnorm

    x, res, w, dy, dh = (t.cuda() for t in _make(4, 64, BF16, BF16, 0.0))
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y, h = add_rmsnorm(xg, res, wg)
    gx, gw = torch.autograd.grad(h, (xg, wg), dh)
    assert torch.equal(gx, dh) and torch.equal(gw, torch.zeros_like(w))
    y, h = add_rmsnorm(x, res, wg)
    (gw,) = torch.autograd.grad(y, wg, dy)
    ref = fwd_bwd(x.cpu(), res.cpu(), w.cpu(), dy.cpu(), None, 1e-6, 0.0)
    _within(gw, ref.dw, ref.dw_terms, 200, "dw")


@pytest.mark.gpu
def test_leading_dimensions_and_nothing_to_do():
    from kernels.rmsnorm import add_rmsnorm, add_rmsnorm_int8

    w = torch.ones(64, device="cuda", dtype=BF16, requires_grad=True)
    x = torch.randn(2, 3, 5, 64, device="cuda").to(BF16).requires_grad_(True)
    y, h = add_rmsnorm(x, x, w)
    y2, h2 = add_rmsnorm(x.view(30, 64), x.view(30, 64), w)
    assert torch.equal(y.view(30, 64), y2) and torch.equal(h.view(30, 64), h2)
    xt = x.detach().transpose(0, 2)
    assert torch.equal(add_rmsnorm(xt, xt, w)[0], y.transpose(0, 2))
    z = torch.zeros(0, 64, device="cuda", dtype=BF16, requires_grad=True)
    y, h = add_rmsnorm(z, z, w)
    assert y.shape == (0, 64) and torch.equal(torch.autograd.grad(y, w, torch.zeros_like(y))[0], torch.zeros_like(w))
    rows, h = add_rmsnorm_int8(z.detach(), z.detach(), w.detach())
    assert rows.values.shape == (0, 64) and rows.dequantize().shape == (0, 64)
    y, _ = add_rmsnorm(x.detach()[0, 0, 0], None, w)  # one row
    assert y.shape == (64,)


# ---------------------------------------------------------------------------
# 8 bits
# ---------------------------------------------------------------------------
def _check8(x, res, w, offset, eps=1e-6):
    from kernels.rmsnorm import add_rmsnorm_int8

    ref = fwd_bwd(x, res, w, None, None, eps, offset)
    q, unit = quantize(ref.h.double() * (w.double() + offset))
    rows, h = add_rmsnorm_int8(_gpu(x), None if res is None else _gpu(res), w.cuda(), eps=eps, offset=offset)
    assert torch.equal(h.cpu(), ref.h)
    assert rows.values.dtype == torch.int8 and rows.dtype == x.dtype
    assert torch.equal(rows.values.cpu().to(torch.int64), q)
    assert bool((rows.padded[:, x.shape[1]:] == 0).all())
    s = unit * ref.rstd
    torch.testing.assert_close(rows.scale.cpu().double(), s, rtol=(400 if x.shape[1] > 4096 else 100) * U, atol=1e-38)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,w_dtype,offset", [(BF16, BF16, 0.0), (BF16, BF16, 1.0), (FP16, FP16, 0.0), (FP16, FP32, 0.0),
                                                  (FP32, FP32, 0.0), (FP32, BF16, 1.0)])
@pytest.mark.parametrize("rows,H", [(1, 1), (5, 13), (300, 700), (40, 4096), (3, 5001), (2, 17000)])
def test_int8_rows(rows, H, dtype, w_dtype, offset):
    x, res, w, _, _ = _make(rows, H, dtype, w_dtype, offset, seed=rows + H, pad=3)
    _check8(x, res, w, offset)
    _check8(x, None, w, offset)


@pytest.mark.gpu
def test_int8_borders():
    """Values that lie on a border between two integers, and next to one."""
    k = torch.arange(0, 127).float()
    row = torch.cat([k + 0.5, -(k + 0.5), torch.tensor([127.0])]).to(FP32)
    near = torch.stack([row, torch.nextafter(row, torch.full_like(row, 1e9)), torch.nextafter(row, torch.full_like(row, -1e9))])
    near[:, -1] = 127.0
    near = near.clamp(-127, 127)
    _check8(near, None, torch.ones(row.numel()), 0.0)
    _check8((near * 3.7).float(), None, torch.full((row.numel(),), 1.1), 0.0)
    _check8(near.to(BF16), None, torch.ones(row.numel(), dtype=BF16), 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-20, 1e18])
def test_int8_magnitudes(scale):
    from kernels.int8 import quantize_int8_rows

    g = torch.Generator().manual_seed(3)
    x = (torch.randn(6, 300, generator=g) * scale).float()
    q, unit = quantize(x)
    rows = quantize_int8_rows(x.cuda())
    assert torch.equal(rows.values.cpu().to(torch.int64), q)
    torch.testing.assert_close(rows.scale.cpu().double(), unit, rtol=4 * U, atol=2.0 ** -149)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_int8_zeros_and_not_finite(dtype):
    from kernels.rmsnorm import add_rmsnorm_int8

    x = torch.randn(6, 100).to(dtype)
    x[1] = 0
    x[2, 7] = float("inf")
    x[3, 99] = float("nan")
    x[4, 0] = float("-inf")
    zero = torch.zeros_like(x)
    rows, h = add_rmsnorm_int8(x.cuda(), zero.cuda(), torch.ones(100, dtype=dtype).cuda())
    assert rows.scale[1] == 0 and bool((rows.values[1] == 0).all())
    for r in range(6):
        assert bool(torch.isnan(rows.scale[r])) == (r in (2, 3, 4))
        assert bool(torch.isnan(rows.dequantize()[r]).all()) == (r in (2, 3, 4))


def test_refusals():
    from kernels.rmsnorm import add_rmsnorm, add_rmsnorm_int8

    x, w = torch.zeros(2, 8), torch.zeros(8)
    for f in (add_rmsnorm, add_rmsnorm_int8):
        with pytest.raises(ValueError, match="weight"):
            f(x, x, w[:7])
        with pytest.raises(ValueError, match="residual"):
            f(x, x[:1], w)
        with pytest.raises(TypeError, match="same dtype"):
            f(x, x.half(), w)
        with pytest.raises(TypeError, match="fp16, bf16 or fp32"):
            f(x.double(), x.double(), w)
        for eps in (-1e-6, float("nan")):
            with pytest.raises(ValueError, match="eps"):
                f(x, x, w, eps=eps)
        with pytest.raises(RuntimeError, match="GPU"):
            f(x, x, w)


@pytest.mark.gpu
def test_int8_refuses_a_lost_gradient():
    from kernels.rmsnorm import add_rmsnorm_int8

    x = torch.zeros(2, 8, device="cuda")
    with pytest.raises(ValueError, match="no gradient"):
        add_rmsnorm_int8(x.requires_grad_(True), None, torch.zeros(8, device="cuda"))
    with torch.no_grad():
        add_rmsnorm_int8(x, None, torch.zeros(8, device="cuda"))


def test_entry_point_refusals():
    from forge_hip import _lib as L

    def fwd(dtype=2, wd=2, x=16, ldx=8, res=16, ldr=8, w=16, h=16, y=16, rows=2, H=8):
        return L.forge_add_rmsnorm_fwd(dtype, wd, x, ldx, res, ldr, w, h, y, None, rows, H, 1e-6, 0.0, None)

    assert fwd(dtype=3) == 2 and fwd(wd=9) == 2
    assert fwd(rows=-1) == 1 and fwd(H=-1) == 1 and fwd(ldx=7) == 1 and fwd(ldr=7) == 1
    assert fwd(x=None) == 1 and fwd(w=None) == 1 and fwd(h=None) == 1 and fwd(y=None) == 1
    assert fwd(rows=0, x=None, res=None, w=None, h=None, y=None) == 0

    def q8(q=16, ldq=16, scale=16):
        return L.forge_add_rmsnorm_int8(2, 2, 16, 8, None, 0, 16, None, q, ldq, scale, 2, 8, 1e-6, 0.0, None)

    assert q8(ldq=8) == 1 and q8(ldq=24) == 1 and q8(q=24) == 1 and q8(scale=None) == 1 and q8(q=None) == 1

    def bwd(dy=16, dh=16, h=16, w=16, rstd=16, d=16, dw=16, work=16, ld=8, dtype=2):
        return L.forge_add_rmsnorm_bwd(dtype, 2, dy, ld, dh, ld, h, ld, w, rstd, d, dw, work, 2, 8, 0.0, None)

    assert bwd(ld=7) == 1 and bwd(dtype=3) == 2
    for n in ("dy", "h", "w", "rstd", "d", "work"):
        assert bwd(**{n: None}) == 1, n
    assert L.forge_add_rmsnorm_bwd_workspace(2, 100, 64) == 25 * 64 * 4
    assert L.forge_add_rmsnorm_bwd_workspace(2, -1, 64) == -1


@pytest.mark.gpu
def test_gradients_are_tensors_of_their_own():
    """x's and the residual's gradient are the same values: changing one's in place leaves the other's."""
    from kernels.rmsnorm import add_rmsnorm

    x, r, w = (torch.randn(*s, device="cuda").requires_grad_(True) for s in ((5, 64), (5, 64), (64,)))
    y, h = add_rmsnorm(x, r, w)
    (y.sum() + h.sum()).backward()
    before = r.grad.clone()
    assert torch.equal(x.grad, before)
    x.grad.zero_()
    assert torch.equal(r.grad, before)
    # one tensor for both
    x.grad = None
    y, h = add_rmsnorm(x, x, w)
    (y.sum() + h.sum()).backward()
    d = x.grad.clone()
    a, b = x.detach().clone().requires_grad_(True), x.detach().clone().requires_grad_(True)
    y, h = add_rmsnorm(a, b, w)
    (y.sum() + h.sum()).backward()
    assert torch.equal(d, a.grad + b.grad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,H", [(FP32, 3), (BF16, 7), (FP16, 8), (FP32, 4), (BF16, 9), (BF16, 8191), (FP32, 8191), (BF16, 16377)])
def test_rows_about_a_vector_and_about_each_kernel(dtype, H):
    _check(37, H, dtype, dtype, pad=3)
    x, res, w, _, _ = _make(37, H, dtype, dtype, 0.0, pad=3)
    _check8(x, res, w, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("H", [3, 520, 2305, 20001])
@pytest.mark.parametrize("size,eps", [(1e-16, 0.0), (1e-13, 0.0), (1e13, 1e-6), (1e15, 1e-6), (1e16, 1e-6)])
def test_gradients_of_rows_of_any_size(size, eps, H, dtype):
    """Rows whose rstd has no cube in fp32 (rstd 1e13: infinite, 1e-15: a subnormal of one bit)."""
    from kernels.rmsnorm import add_rmsnorm

    x, res, w, dy, _ = _make(5, H, dtype, dtype, 0.0, seed=H)
    x, res = ((t.double() * size).to(dtype) for t in (x, res))
    ref = fwd_bwd(x, res, w, dy, None, eps, 0.0)
    leaves = [t.cuda().requires_grad_(True) for t in (x, res, w)]
    got = torch.autograd.grad(add_rmsnorm(*leaves, eps=eps)[0], leaves, dy.cuda())
    k = 400 if H > 4096 else 100
    for t in got[:2]:
        _within(t, ref.d, ref.d_terms, 2 * k, "d")
    _within(got[2], ref.dw, ref.dw_terms, 181, "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e30, 1e36, 1e38])
@pytest.mark.parametrize("H", [64, 5001])
def test_int8_scales_of_large_weights(size, H):
    """a rstd / 127 is finite where a rstd is not."""
    x = torch.full((3, H), 1e-3)
    x[:, :2] = torch.tensor([1.0, -0.5])
    _check8(x, None, torch.full((H,), size), 0.0)


@pytest.mark.gpu
def test_rows_without_columns():
    from kernels.rmsnorm import add_rmsnorm, add_rmsnorm_int8

    w = torch.ones(0, device="cuda", requires_grad=True)
    x = torch.zeros(2, 3, 0, device="cuda", requires_grad=True)
    y, h = add_rmsnorm(x, x, w)
    assert y.shape == h.shape == (2, 3, 0)
    assert [g.shape for g in torch.autograd.grad((y, h), (x, w), (y, h))] == [(2, 3, 0), (0,)]
    rows, h = add_rmsnorm_int8(x.detach(), None, w.detach())
    assert rows.values.shape == (2, 3, 0) and rows.scale.shape == (6,)
