"""Linear layers on frozen 8-bit weights (`int8_linear`).

Tolerances, derived before the first run: the integers and their sum are exact, so a
result has the rounding of the sum to fp32, three of the scales and their products,
one of the bias's addition (6 roundings of 2^-24 of the terms), and that of its type."""
import pytest
import torch

from oracle.int8 import linear, quantize

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _within(got, ref, terms, k, what):
    f = torch.finfo(got.dtype)
    bound = ref.abs() * (f.eps / 2) + terms * (k * U * (1 + f.eps)) + f.smallest_normal * f.eps
    over = (got.detach().double().cpu() - ref).abs() - bound
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, f"{what}: off by {worst:.3e} more than the bound"


def _weight(n, k, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, (n, k), generator=g).to(torch.int8), torch.rand(n, generator=g) * 0.02 + 0.001


def _check(m, n, k, dtype, bias=False, train=True, out_dtype=None, seed=0):
    from kernels.int8 import Int8Weight, int8_linear

    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(dtype)
    w, ws = _weight(n, k)
    b = torch.randn(n, generator=g).to(out_dtype or dtype) if bias else None
    weight = Int8Weight(w.cuda(), ws.cuda(), backward=train)
    xg = x.cuda().requires_grad_(train)
    y = int8_linear(xg, weight, None if b is None else b.cuda(), out_dtype=out_dtype)
    assert y.dtype == (out_dtype or dtype)
    ref, terms = linear(*quantize(x), w, ws, b)
    _within(y, ref, terms, 6, "y")
    if train:
        dy = torch.randn(m, n, generator=g).to(y.dtype)
        (dx,) = torch.autograd.grad(y, xg, dy.cuda())
        ref, terms = linear(*quantize(dy.double() * ws.double()), w.T, torch.ones(k))
        _within(dx, ref, terms, 6, "dx")
        # the gradient of the formula, up to the rounding of dy w_scale to 8 bits: at most half a unit each
        full = (dy.double() * ws.double()) @ w.double()
        unit = quantize(dy.double() * ws.double())[1]
        slack = 0.5 * unit.unsqueeze(1) * w.double().abs().sum(0)
        assert bool(((dx.double().cpu() - full).abs() <= slack + full.abs() * torch.finfo(dtype).eps + 1e-30).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 130, 500), (16, 1024, 512), (17, 33, 100), (32, 2017, 1003), (33, 70, 64),
                                   (100, 1024, 4096), (333, 257, 130), (129, 640, 4101), (64, 4096, 300), (20, 9001, 200),
                                   (70, 70, 14336)])
def test_sizes(m, n, k, dtype):
    _check(m, n, k, dtype, bias=m % 2 == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("m,n,k", [(2600, 3000, 300), (4096, 2048, 1024), (1500, 1504, 77), (2049, 4104, 48)])
def test_large_tiles(m, n, k, dtype):
    _check(m, n, k, dtype, bias=True)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_output_types(m):
    for dtype in (BF16, FP16, FP32):
        for out in (BF16, FP16, FP32):
            _check(m, 96, 160, dtype, bias=True, out_dtype=out)


@pytest.mark.gpu
def test_the_largest_sum():
    """K = 2^17 of the largest products: 2^31 - ..., just inside 32 bits."""
    from kernels.int8 import Int8Weight, int8_linear

    k = 1 << 17
    w = torch.full((3, k), 127, dtype=torch.int8)
    w[1] = -127
    x = torch.ones(2, k, device="cuda")
    y = int8_linear(x, Int8Weight(w.cuda(), torch.ones(3, device="cuda")), out_dtype=FP32)
    ref = torch.tensor([127.0, -127.0, 127.0], dtype=torch.float64) * k
    assert bool(((y.double().cpu() - ref).abs() <= ref.abs() * 6 * U).all())


@pytest.mark.gpu
def test_rows_from_the_norm_and_quantizer():
    from kernels.int8 import Int8Weight, int8_linear, quantize_int8_rows
    from kernels.rmsnorm import add_rmsnorm_int8

    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 7, 300, generator=g).to(BF16).cuda()
    w, ws = _weight(96, 300)
    weight = Int8Weight(w.cuda(), ws.cuda())
    y = int8_linear(x, weight)
    assert y.shape == (3, 7, 96) and torch.equal(y, int8_linear(quantize_int8_rows(x), weight))
    assert torch.equal(quantize_int8_rows(x).values.cpu().long(), quantize(x.cpu())[0])
    rows, h = add_rmsnorm_int8(x, x, torch.ones(300, device="cuda", dtype=BF16))
    y = int8_linear(rows, weight, out_dtype=FP32)
    assert y.shape == (3, 7, 96)
    ref, terms = linear(rows.padded[:, :300].cpu(), rows.scale.cpu(), w, ws)
    _within(y.view(21, 96), ref, terms, 6, "y")
    one = x[0, 0]
    assert torch.equal(int8_linear(one, weight), int8_linear(x, weight)[0, 0])
    assert torch.equal(quantize_int8_rows(one).values, quantize_int8_rows(x).values[0, 0])


@pytest.mark.gpu
def test_weights_from_floats():
    from kernels.int8 import Int8Weight

    g = torch.Generator().manual_seed(6)
    w = torch.randn(70, 130, generator=g).to(BF16)
    q, s = quantize(w)
    weight = Int8Weight.from_float(w.cuda(), backward=True)
    assert torch.equal(weight.values.cpu().long(), q)
    torch.testing.assert_close(weight.scale.cpu().double(), s, rtol=4 * U, atol=0)
    assert torch.equal(weight.transposed[:, :70], weight.values.t()) and bool((weight.transposed[:, 70:] == 0).all())
    torch.testing.assert_close(weight.dequantize().cpu().double(), q * s.unsqueeze(1), rtol=1e-6, atol=0)


@pytest.mark.gpu
def test_not_finite_rows_and_nothing_to_do():
    from kernels.int8 import Int8Weight, int8_linear

    w, ws = _weight(40, 64)
    weight = Int8Weight(w.cuda(), ws.cuda(), backward=True)
    x = torch.randn(5, 64, device="cuda")
    x[1, 3] = float("nan")
    x[2, 5] = float("-inf")
    x[3] = 0
    y = int8_linear(x, weight)
    assert bool(torch.isnan(y[1:3]).all()) and bool((y[3] == 0).all()) and bool(torch.isfinite(y[[0, 3, 4]]).all())
    z = torch.zeros(0, 64, device="cuda", requires_grad=True)
    out = int8_linear(z, weight)
    assert out.shape == (0, 40) and torch.autograd.grad(out, z, torch.zeros_like(out))[0].shape == (0, 64)
    # no columns, no channels
    empty = Int8Weight(torch.zeros(3, 0, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"))
    b = torch.arange(3.0, device="cuda")
    assert torch.equal(int8_linear(torch.zeros(2, 0, device="cuda"), empty, b), b.expand(2, 3))
    none = Int8Weight(torch.zeros(0, 64, dtype=torch.int8, device="cuda"), torch.ones(0, device="cuda"))
    assert int8_linear(x, none).shape == (5, 0)


@pytest.mark.gpu
def test_strided_inputs():
    from kernels.int8 import Int8Weight, int8_linear

    w, ws = _weight(40, 64)
    weight = Int8Weight(w.cuda(), ws.cuda(), backward=True)
    wide = torch.randn(9, 131, device="cuda").to(BF16)
    for x in (wide[:, 1:65], wide[:, ::2][:, :64], wide[0, :64].expand(9, 64), wide[:, :64].t().contiguous().t()):
        y = int8_linear(x, weight)
        assert torch.equal(y, int8_linear(x.contiguous(), weight))
        xg = x.detach().requires_grad_(True)
        dy = torch.randn(40, 9, device="cuda").to(BF16).t()
        got = torch.autograd.grad(int8_linear(xg, weight), xg, dy)[0]
        xc = x.contiguous().detach().requires_grad_(True)
        assert torch.equal(got, torch.autograd.grad(int8_linear(xc, weight), xc, dy.contiguous())[0])


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    from kernels.int8 import Int8Weight, int8_linear, quantize_int8_rows

    w, ws = _weight(40, 64)
    weight = Int8Weight(w.cuda(), ws.cuda())
    x = torch.zeros(2, 64, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="backward=True"):
        int8_linear(x, weight)
    with pytest.raises(ValueError, match="no gradient"):
        quantize_int8_rows(x)
    x = x.detach()
    with pytest.raises(ValueError, match="columns"):
        int8_linear(x[:, :63], weight)
    with pytest.raises(ValueError, match="frozen"):
        int8_linear(x, weight, torch.zeros(40, device="cuda", requires_grad=True))
    with pytest.raises(ValueError, match="bias"):
        int8_linear(x, weight, torch.zeros(39, device="cuda"))
    with pytest.raises(TypeError, match="out_dtype"):
        int8_linear(x, weight, out_dtype=torch.float64)
    with pytest.raises(TypeError, match="Int8Weight"):
        int8_linear(x, w.cuda())
    with pytest.raises(TypeError, match="fp16, bf16 or fp32"):
        int8_linear(x.double(), weight)


def test_refusals():
    from kernels.int8 import Int8Weight, quantize_int8_rows

    w, ws = _weight(4, 8)
    with pytest.raises(ValueError, match="int8 matrix"):
        Int8Weight(w.float(), ws)
    with pytest.raises(ValueError, match="scale"):
        Int8Weight(w, ws[:3])
    with pytest.raises(ValueError, match="32 bits"):
        Int8Weight(torch.zeros(1, (1 << 17) + 1, dtype=torch.int8), ws[:1])
    with pytest.raises(RuntimeError, match="GPU"):
        Int8Weight(w, ws)
    with pytest.raises(RuntimeError, match="GPU"):
        quantize_int8_rows(torch.zeros(2, 8))


def test_entry_point_refusals():
    from forge_hip import _lib as L

    def gemm(a=16, lda=64, rs=16, b=16, ldb=64, cs=16, c=16, ldc=40, dtype=2, M=4, N=40, K=64):
        return L.forge_int8_gemm(a, lda, rs, b, ldb, cs, None, c, ldc, dtype, M, N, K, None, None)

    assert gemm(dtype=3) == 2
    for kw in ({"M": -1}, {"K": (1 << 17) + 1}, {"lda": 48}, {"ldb": 72}, {"lda": 1 << 22}, {"a": 24}, {"b": 8}, {"ldc": 39},
               {"a": None}, {"b": None}, {"rs": None}, {"cs": None}, {"c": None}):
        assert gemm(**kw) == 1, kw
    assert gemm(M=0, a=None, c=None) == 0
    # a product that is split over K needs its workspace
    assert L.forge_int8_gemm_workspace(4, 40, 64) == 0 and L.forge_int8_gemm_workspace(100, 1024, 14336) == 8 * 100 * 1024 * 4
    assert gemm(M=100, N=1024, K=14336, lda=14336, ldb=14336, ldc=1024) == 1 and b"work" in L.forge_last_error()
    assert L.forge_int8_gemm_workspace(-1, 40, 64) == -1
    def linear(x=16, ldx=64, w=16, c=16, work=16, M=4, N=40, K=64):
        return L.forge_int8_linear(2, x, ldx, None, w, 64, 16, None, c, N, 2, M, N, K, work, None)

    assert L.forge_int8_linear_workspace(4, 40, 60) == 4 * 64 + 16 and L.forge_int8_linear_workspace(-1, 40, 64) == -1
    assert linear(M=0, x=None, work=None) == 0 and linear(work=None) == 1 and linear(work=24) == 1
    assert linear(M=-1) == 1 and linear(ldx=63) == 1 and linear(x=None) == 1
    assert L.forge_transpose_1b(None, 8, 4, 8, 16, 16, None) == 1
    assert L.forge_transpose_1b(16, 7, 4, 8, 16, 16, None) == 1
    assert L.forge_quantize_rows(2, 16, 8, None, 16, 8, 16, 2, 8, None) == 1


# sizes of each engine: rows, tiles in parts of K, both kinds of tiles, large tiles with and without aligned rows
_ENGINES = [(4, 64, 64), (50, 1024, 512), (100, 1024, 4096), (333, 257, 130), (1000, 4096, 128), (2600, 3000, 300),
            (2600, 3001, 48)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (FP32, FP32), (FP32, FP16)])
@pytest.mark.parametrize("m,n,k", _ENGINES)
def test_sums_times_one_scale_past_the_largest_value(m, n, k, dtype, out_dtype):
    """Rows of 1e35 and weights of 1e-33, rows of 1e-30 and weights of 1e30 beside rows of usual size: the products
    of the integers and one of the scales are past fp32's range, or below it, and the results are not."""
    from kernels.int8 import Int8Weight, int8_linear

    g = torch.Generator().manual_seed(m)
    rows = torch.ones(m, 1)
    w, ws = _weight(n, k)
    for large in (True, False):
        rows[::3] = 1e35 if large else 1e-30
        x = (torch.randn(m, k, generator=g) * rows).to(dtype)
        scale = ws * (1e-33 if large else 1e30)
        if not large:
            x[1::3], x[2::3] = x[1::3] * 1e-29, x[2::3] * 0
        b = torch.randn(n, generator=g).to(out_dtype)
        ref, terms = linear(*quantize(x), w, scale, b)
        y = int8_linear(x.cuda(), Int8Weight(w.cuda(), scale.cuda()), b.cuda(), out_dtype=out_dtype)
        if out_dtype == FP16:  # (what passes the type's own largest value is infinite)
            over = ref.abs() >= 65520
            near = (ref.abs() - 65520).abs() < 1
            assert torch.equal(torch.isinf(y.cpu())[~near], over[~near])
            y, ref, terms = y.cpu()[~over & ~near], ref[~over & ~near], terms[~over & ~near]
        _within(y, ref, terms, 6, "y")
    # scales that are not finite, and products of 0 with a large scale
    x = torch.randn(m, k, generator=g)
    x[0] = 3e38
    scale = ws.clone()
    scale[0], scale[-1] = 3e38, float("nan")
    w[0] = 0
    y = int8_linear(x.cuda(), Int8Weight(w.cuda(), scale.cuda()), out_dtype=FP32)
    assert bool(y[:, -1].isnan().all()) and (n == 1 or bool((y[:, 0] == 0).all()))


@pytest.mark.gpu
def test_a_weight_is_a_copy():
    """Values and scales that are changed in place afterwards, also between a forward and its backward."""
    from kernels.int8 import Int8Weight, int8_linear

    w, ws = (t.cuda() for t in _weight(40, 64))
    for scale in (ws, torch.stack([ws, ws], 1)[:, 0]):  # contiguous or not
        values, scale = w.clone(), scale.clone() if scale.is_contiguous() else scale
        weight = Int8Weight(values, scale, backward=True)
        x = torch.randn(3, 64, device="cuda", requires_grad=True)
        y = int8_linear(x, weight)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
        values.zero_()
        scale.zero_()
        assert torch.equal(int8_linear(x, weight), y)
        assert torch.equal(torch.autograd.grad(y, x, torch.ones_like(y))[0], dx)


@pytest.mark.gpu
@pytest.mark.parametrize("bias_dtype", [FP32, BF16, FP16, torch.float64])
@pytest.mark.parametrize("m,n,k", _ENGINES)
def test_a_bias_of_another_type(m, n, k, bias_dtype):
    """Added as it is: only the sum is rounded to the output's type."""
    from kernels.int8 import Int8Weight, int8_linear, quantize_int8_rows

    g = torch.Generator().manual_seed(n)
    w, ws = _weight(n, k)
    b = (torch.randn(n, generator=g, dtype=torch.float64) * 3).to(bias_dtype)
    weight = Int8Weight(w.cuda(), ws.cuda(), backward=True)
    for dtype in (BF16, FP16, FP32):
        x = torch.randn(m, k, generator=g).to(dtype)
        ref, terms = linear(*quantize(x), w, ws, b)
        y = int8_linear(x.cuda(), weight, b.cuda())
        _within(y, ref, terms, 7, "y")  # (a float64 bias: its rounding to fp32 besides)
        assert torch.equal(int8_linear(quantize_int8_rows(x.cuda()), weight, b.cuda()), y)
        assert torch.equal(int8_linear(x.cuda().requires_grad_(True), weight, b.cuda()), y)


def test_entry_points_with_a_bias_type():
    from forge_hip import _lib as L

    def gemm(bias=16, bias_dtype=0, K=64):
        return L.forge_int8_gemm_typed(16, 64, 16, 16, 64, 16, bias, bias_dtype, 16, 40, 2, 4, 40, K, None, None)

    def lin(bias=16, bias_dtype=0, x=16):
        return L.forge_int8_linear_typed(2, x, 64, None, 16, 64, 16, bias, bias_dtype, 16, 40, 2, 4, 40, 64, 16, None)

    assert gemm(bias_dtype=3) == 2 and gemm(bias_dtype=-1) == 2 and b"bias" in L.forge_last_error()
    assert lin(bias_dtype=3) == 2 and b"bias" in L.forge_last_error()
    assert gemm(bias=None, bias_dtype=3, K=-1) == 1 and lin(bias=None, bias_dtype=3, x=None) == 1


def test_rows_that_the_kernels_cannot_read_are_refused():
    from kernels.int8 import Int8Rows

    q, s = torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6)
    assert Int8Rows(q, s, (2, 3, 20), BF16).values.shape == (2, 3, 20)
    for padded, scale, shape in ((q.float(), s, (6, 20)), (q[0], s, (6, 20)), (q, s.double(), (6, 20)), (q, s.half(), (6, 20)),
                                 (q, s[:5], (6, 20)), (q, s.view(6, 1), (6, 20)), (q, s, (5, 20)), (q, s, (2, 4, 20)),
                                 (q, s, (6, 40)), (q, s, ()), (q[:, :24], s, (6, 20)), (q[:, 1:17], s, (6, 16)),
                                 (torch.zeros(6, 24, dtype=torch.int8), s, (6, 20)), (q, torch.zeros(12)[::2], (6, 20)),
                                 (q, s.to("meta"), (6, 20)), (q.t(), torch.zeros(32), (32, 6))):
        with pytest.raises(ValueError, match="Int8Rows"):
            Int8Rows(padded, scale, shape, BF16)
    with pytest.raises(TypeError, match="fp16, bf16 or fp32"):
        Int8Rows(q, s, (6, 20), torch.float64)


@pytest.mark.gpu
def test_no_columns_and_no_channels_with_leading_dimensions():
    from kernels.int8 import Int8Weight, int8_linear, quantize_int8_rows

    empty = Int8Weight(torch.zeros(3, 0, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"), backward=True)
    b = torch.arange(3.0, device="cuda")
    x = torch.zeros(2, 4, 0, device="cuda", requires_grad=True)
    y = int8_linear(x, empty, b)
    assert torch.equal(y, b.expand(2, 4, 3)) and torch.autograd.grad(y, x, torch.ones_like(y))[0].shape == (2, 4, 0)
    rows = quantize_int8_rows(x.detach())
    assert rows.values.shape == (2, 4, 0) and torch.equal(int8_linear(rows, empty, b), b.expand(2, 4, 3))
    none = Int8Weight(torch.zeros(0, 64, dtype=torch.int8, device="cuda"), torch.ones(0, device="cuda"), backward=True)
    x = torch.randn(2, 4, 64, device="cuda", requires_grad=True)
    y = int8_linear(x, none)
    assert y.shape == (2, 4, 0) and torch.equal(torch.autograd.grad(y, x, torch.ones_like(y))[0], torch.zeros_like(x))
    one = torch.zeros(0, device="cuda")
    assert torch.equal(int8_linear(one, empty, b), b)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 50, 300])
def test_more_channels_than_a_gradient_can_sum(m):
    """More than 2^17 channels (an output layer's vocabulary): a product sums over the columns, only the gradient over
    the channels."""
    _check(m, (1 << 17) + 37, 48, BF16, bias=True, train=False)


def test_a_gradient_over_too_many_channels_is_refused():
    from kernels.int8 import Int8Weight

    n = (1 << 17) + 1
    with pytest.raises(ValueError, match="32 bits"):
        Int8Weight(torch.zeros(n, 1, dtype=torch.int8), torch.zeros(n), backward=True)
    with pytest.raises(RuntimeError, match="GPU"):
        Int8Weight(torch.zeros(n, 1, dtype=torch.int8), torch.zeros(n))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", _ENGINES)
def test_large_scales_that_are_negative(m, n, k):
    """Of rows and of channels, where a caller's have signs: as large ones, and 0 times the largest is 0."""
    from kernels.int8 import Int8Rows, Int8Weight, int8_linear

    g = torch.Generator().manual_seed(m)
    w, ws = _weight(n, k)
    pitch = (k + 15) // 16 * 16
    q = torch.randint(-127, 128, (m, pitch), generator=g).to(torch.int8)
    q[:, k:] = 0
    q[1 % m] = 0
    scale = torch.rand(m, generator=g) + 0.5
    scale[::2] *= -1e34
    scale[1 % m] = -1e36
    ws = ws * 1e-33
    ws[::3] *= -1
    ws[-1] = -3e38
    y = int8_linear(Int8Rows(q.cuda(), scale.cuda(), (m, k), FP32), Int8Weight(w.cuda(), ws.cuda())).cpu()
    ref, terms = linear(q[:, :k], scale, w, ws)
    over = ref.abs() > 3.4e38
    assert bool((y[1 % m] == 0).all()) and torch.equal(torch.isinf(y), over)
    _within(y[~over], ref[~over], terms[~over], 6, "y")
