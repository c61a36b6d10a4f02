"""Linear layers on frozen weights of 8-bit integers (csrc/int8_gemm.hip,
csrc/add_rmsnorm.hip).

Weights have a scale for each output channel, activations one for each token
that is found as they come:

    q = round(127 x / a), a = max |x| of the row,  scale = a / 127
    y = (sum_k q[m, k] w[n, k]) scale[m] w_scale[n] + bias[n]

The integers are those of exact arithmetic (half to even) and their sum is exact.  y is
formed of it in fp32 (the sum, its product with a scale, and that with the other plus
the bias are rounded) and then rounded to its type.  A row with an infinity or NaN has a NaN scale, so all that is
computed of it is NaN; a row of zeros has scale 0.

Weights are frozen: there is no gradient for them or the bias.  The gradient of x
is the product with the same integers, of the incoming gradient rounded in the
same way: e = dy w_scale, quantized by rows, times the transposed weight.
"""
from __future__ import annotations

import math
from typing import Optional, Union

import torch

from forge_hip import _lib as L

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
MAX_K = 1 << 17  # where a sum of products still fits 32 bits


def _pitch(k: int) -> int:
    return (k + 15) // 16 * 16


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, K] with a unit stride in K."""
    x2 = x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    if x2.is_contiguous():
        return x2
    if x2.stride(-1) != 1 and x2.shape[-1] > 1 or (x2.shape[0] > 1 and x2.stride(0) < x2.shape[-1]):
        x2 = x2.contiguous()
    return x2


def _ld(x2: torch.Tensor) -> int:
    return max(x2.stride(0), x2.shape[1]) if x2.shape[0] > 1 else x2.shape[1]


class Int8Rows:
    """Rows in 8 bits: `padded` [rows, pitch] (K to the next multiple of 16 or more, zeros
    behind K), `scale` [rows] in fp32, the shape and type of what they stand for."""

    __slots__ = ("padded", "scale", "shape", "dtype")

    def __init__(self, padded: torch.Tensor, scale: torch.Tensor, shape, dtype: torch.dtype):
        shape = torch.Size(shape)
        if dtype not in _DTYPES:
            raise TypeError(f"Int8Rows stand for fp16, bf16 or fp32, got {dtype}")
        rows = math.prod(shape[:-1])
        if (len(shape) < 1 or padded.dim() != 2 or padded.dtype != torch.int8 or not padded.is_contiguous()
                or padded.shape[0] != rows or padded.shape[1] < shape[-1] or padded.shape[1] % 16):
            raise ValueError(f"Int8Rows of {tuple(shape)} need contiguous int8 rows of a multiple of 16 columns, got "
                             f"{padded.dtype} {tuple(padded.shape)}")
        if scale.shape != (rows,) or scale.dtype != torch.float32 or not scale.is_contiguous() or scale.device != padded.device:
            raise ValueError(f"Int8Rows need contiguous fp32 scales [{rows}] on {padded.device}, got {scale.dtype} "
                             f"{tuple(scale.shape)} on {scale.device}")
        self.padded, self.scale, self.shape, self.dtype = padded, scale, shape, dtype

    @classmethod
    def _of(cls, padded, scale, shape, dtype) -> "Int8Rows":
        """Of this package's own making: without the checks."""
        self = cls.__new__(cls)
        self.padded, self.scale, self.shape, self.dtype = padded, scale, shape, dtype
        return self

    @property
    def values(self) -> torch.Tensor:
        """The integers, in `shape`."""
        return self.padded[:, :self.shape[-1]].unflatten(0, self.shape[:-1]) if len(self.shape) > 1 else self.padded[0, :self.shape[0]]

    def dequantize(self) -> torch.Tensor:
        """What the rows stand for, in fp32."""
        return (self.padded[:, :self.shape[-1]].float() * self.scale.unsqueeze(1)).reshape(self.shape)


def _new_rows(rows: int, k: int, device):
    return torch.empty(rows, _pitch(k), dtype=torch.int8, device=device), torch.empty(rows, dtype=torch.float32, device=device)


def _quantize(x2: torch.Tensor, col_scale: Optional[torch.Tensor] = None):
    q, scale = _new_rows(x2.shape[0], x2.shape[1], x2.device)
    if x2.shape[1] == 0:
        return q, scale.zero_()
    if x2.shape[0]:
        with L.on_device(x2):
            L.check(L.forge_quantize_rows(L.dtype_code(x2.dtype), x2.data_ptr(), _ld(x2), L.ptr(col_scale), q.data_ptr(),
                                          q.shape[1], scale.data_ptr(), x2.shape[0], x2.shape[1], L.stream_of(x2)),
                    "forge_quantize_rows")
    return q, scale


def _check_float(x, what):
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what} must be fp16, bf16 or fp32, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError(f"{what} must have at least one dimension")
    L.require_gpu(x)


def quantize_int8_rows(x: torch.Tensor) -> Int8Rows:
    """The rows of x [..., K] in 8 bits with a scale each.  Not differentiable
    (int8_linear is): raises where a gradient would be lost."""
    _check_float(x, "x")
    if torch.is_grad_enabled() and x.requires_grad:
        raise ValueError("quantize_int8_rows has no gradient; pass x itself to int8_linear, or a detached x")
    L.refuse_tangents(x)
    return Int8Rows._of(*_quantize(_rows(x)), x.shape, x.dtype)


def _check_sums(shape, backward):
    """A product sums over the columns, the gradient of x over the channels."""
    if shape[1] > MAX_K or (backward and shape[0] > MAX_K):
        raise ValueError(f"a sum over more than {MAX_K} products does not fit 32 bits, got {tuple(shape)}"
                         + (" with backward=True" if backward else ""))


class Int8Weight:
    """A frozen weight [N, K] of 8-bit integers with a scale for each of its N channels,
    laid out for the kernels (a copy of both).  K up to 2^17.  backward: also its
    transpose, which the gradient of the activations reads; N up to 2^17 then."""

    def __init__(self, values: torch.Tensor, scale: torch.Tensor, *, backward: bool = False):
        if values.dim() != 2 or values.dtype != torch.int8:
            raise ValueError(f"values must be an int8 matrix [N, K], got {values.dtype} {tuple(values.shape)}")
        if scale.shape != values.shape[:1] or scale.dtype != torch.float32:
            raise ValueError(f"scale must be fp32 [{values.shape[0]}], got {scale.dtype} {tuple(scale.shape)}")
        if scale.device != values.device:
            raise ValueError(f"values and scale must be on one device, got {values.device} and {scale.device}")
        n, k = values.shape
        _check_sums(values.shape, backward)
        L.require_gpu(values)
        self.shape = values.shape
        self.padded = torch.zeros(n, _pitch(k), dtype=torch.int8, device=values.device)
        self.padded[:, :k] = values
        self._finish(scale.detach().clone(memory_format=torch.contiguous_format), backward)

    def _finish(self, scale, backward):
        self.scale = scale
        self.transposed = None
        if backward:
            n, k = self.shape
            self.transposed = torch.empty(k, _pitch(n), dtype=torch.int8, device=self.padded.device)
            if n and k:
                with L.on_device(self.padded):
                    L.check(L.forge_transpose_1b(self.padded.data_ptr(), self.padded.shape[1], n, k,
                                                 self.transposed.data_ptr(), self.transposed.shape[1],
                                                 L.stream_of(self.padded)), "forge_transpose_1b")
            self.ones = torch.ones(k, dtype=torch.float32, device=self.padded.device)

    @classmethod
    def from_float(cls, weight: torch.Tensor, *, backward: bool = False) -> "Int8Weight":
        """weight [N, K] rounded by channels, as rows of activations are."""
        _check_float(weight, "weight")
        if weight.dim() != 2:
            raise ValueError(f"weight must be a matrix [N, K], got {tuple(weight.shape)}")
        _check_sums(weight.shape, backward)
        self = cls.__new__(cls)
        self.shape = weight.shape
        self.padded, scale = _quantize(_rows(weight.detach()))
        self._finish(scale, backward)
        return self

    @property
    def values(self) -> torch.Tensor:
        return self.padded[:, :self.shape[1]]

    def dequantize(self) -> torch.Tensor:
        return self.values.float() * self.scale.unsqueeze(1)


def _bias_code(bias):
    return 0 if bias is None else L.dtype_code(bias.dtype)


def _product(q, scale, w, w_scale, bias, dtype, n, k):
    out = torch.empty(q.shape[0], n, dtype=dtype, device=q.device)
    if out.numel():
        nbytes = L.forge_int8_gemm_workspace(q.shape[0], n, k)
        work = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        with L.on_device(q):
            L.check(L.forge_int8_gemm_typed(q.data_ptr(), q.shape[1], scale.data_ptr(), w.data_ptr(), w.shape[1],
                                            w_scale.data_ptr(), L.ptr(bias), _bias_code(bias), out.data_ptr(), n,
                                            L.dtype_code(dtype), q.shape[0], n, k, L.ptr(work), L.stream_of(q)),
                    "forge_int8_gemm")
    return out


def _linear(x2, col_scale, w, w_scale, bias, dtype, n, k):
    """The rows of x2 [M, k] (times col_scale) rounded to 8 bits, times w [n, k]: [M, n]."""
    rows, device = x2.shape[0], x2.device
    out = torch.empty(rows, n, dtype=dtype, device=device)
    if rows and n:
        work = torch.empty(L.forge_int8_linear_workspace(rows, n, k), dtype=torch.uint8, device=device)
        with L.on_device(x2):
            L.check(L.forge_int8_linear_typed(L.dtype_code(x2.dtype), x2.data_ptr(), _ld(x2), L.ptr(col_scale), w.data_ptr(),
                                              w.shape[1], w_scale.data_ptr(), L.ptr(bias), _bias_code(bias), out.data_ptr(),
                                              n, L.dtype_code(dtype), rows, n, k, work.data_ptr(), L.stream_of(x2)),
                    "forge_int8_linear")
    return out


class Int8LinearFunction(torch.autograd.Function):
    """forward(ctx, x, weight, bias, dtype) on checked arguments; keeps nothing of x."""

    @staticmethod
    def forward(ctx, x, weight, bias, dtype):
        ctx.weight, ctx.x_shape, ctx.x_dtype = weight, x.shape, x.dtype
        n, k = weight.shape
        return _linear(_rows(x), None, weight.padded, weight.scale, bias, dtype, n, k).view(*x.shape[:-1], n)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        w = ctx.weight
        n, k = w.shape
        dx = _linear(_rows(dy), w.scale, w.transposed, w.ones, None, ctx.x_dtype, k, n)
        return dx.view(ctx.x_shape), None, None, None


def int8_linear(x: Union[torch.Tensor, Int8Rows], weight: Int8Weight, bias: Optional[torch.Tensor] = None, *,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x [..., K] times weight [N, K], plus bias [N]: [..., N] in out_dtype (default x's type).
    The bias is added in fp32, whatever its type.

    x in fp16, bf16 or fp32 is rounded to 8 bits by rows; Int8Rows
    (quantize_int8_rows, add_rmsnorm_int8) are taken as they are.  A gradient of x
    needs a weight made with backward=True."""
    if not isinstance(weight, Int8Weight):
        raise TypeError(f"weight must be an Int8Weight, got {type(weight).__name__}")
    ready = isinstance(x, Int8Rows)
    if not ready:
        _check_float(x, "x")
    device = x.scale.device if ready else x.device
    n, k = weight.shape
    if x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1]} columns, the weight {k}")
    if weight.scale.device != device:
        raise ValueError(f"weight must be on x's device {device}")
    dtype = x.dtype if out_dtype is None else out_dtype
    if dtype not in _DTYPES:
        raise TypeError(f"out_dtype must be fp16, bf16 or fp32, got {dtype}")
    if bias is not None:
        if bias.shape != (n,) or bias.device != device or not bias.is_floating_point():
            raise ValueError(f"bias must be [{n}] on {device}, got {tuple(bias.shape)} on {bias.device}")
        if torch.is_grad_enabled() and bias.requires_grad:
            raise ValueError("the bias of an int8_linear is frozen; add a trained one to the result")
        L.refuse_tangents(bias)
        bias = (bias if bias.dtype in _DTYPES else bias.float()).contiguous()
    if ready:
        return _product(x.padded, x.scale, weight.padded, weight.scale, bias, dtype, n, k).view(*x.shape[:-1], n)
    if torch.is_grad_enabled() and x.requires_grad:
        if weight.transposed is None:
            raise ValueError("the gradient of x needs a weight made with backward=True")
        return Int8LinearFunction.apply(x, weight, bias, dtype)
    L.refuse_tangents(x)
    return _linear(_rows(x), None, weight.padded, weight.scale, bias, dtype, n, k).view(*x.shape[:-1], n)


__all__ = ["Int8LinearFunction", "Int8Rows", "Int8Weight", "int8_linear", "quantize_int8_rows"]
