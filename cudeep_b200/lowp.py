"""Low-precision and grouped products over `Tensor`: 8-bit floating point with block scales, Linear layers on it, their
backward pass from activations kept in 8 bits, and products of row groups that each have a matrix of their own.

The reference has no counterpart.  Everything goes through the C ABI (include/cudeep_b200.h, "8-bit and grouped products");
errors surface as RuntimeError.  16-bit tensors are bfloat16 here; the C ABI takes float16 as well.

A training step of a layer y = act(x W^T + b) whose activations are kept in 8 bits:

    x8, w8 = quantize_fp8(x), quantize_fp8(w, tiles=True)
    z = linear_fp8(x8, w8, b)                       # the product of the very codes that are kept
    z8 = quantize_fp8(z)
    ...
    dx, dw, db = linear_backward_saved(dy, x8, w, z8, "gelu")
"""
from __future__ import annotations

from typing import Optional

from . import _lib
from .tensor import DType, Tensor, _TYPE_CODE, _epilogue_code

BLOCK = 128     # elements along a row that share a scale


def _code(dtype: DType, what: str) -> int:
    if dtype not in _TYPE_CODE:
        raise RuntimeError(f"{what}: float32 or bfloat16 expected, got {dtype.name}")
    return _TYPE_CODE[dtype]


def _matrix(t, what: str, dtype: Optional[DType] = None) -> Tensor:
    if not isinstance(t, Tensor) or t.ndim() != 2:
        raise RuntimeError(f"{what}: 2-D Tensor expected")
    return _dense(t, what, dtype)


def _dense(t: Tensor, what: str, dtype: Optional[DType] = None) -> Tensor:
    if dtype is not None and t.dtype() != dtype:
        raise RuntimeError(f"{what}: {dtype.name} expected, got {t.dtype().name}")
    if not t.is_contiguous():
        raise RuntimeError(f"{what} requires contiguous tensors")
    return t


def _like(ref: Tensor, shape, dtype: DType) -> Tensor:
    return Tensor(shape, dtype, _stream=ref.stream)


def _ptr(t: Optional[Tensor]):
    return None if t is None else t._storage.ptr


class Fp8Tensor:
    """A matrix as e4m3 codes (`data`) with power-of-two `scales`: one for each 128 columns of a row, laid out
    [column block][row], or with `tiles` one for each block of 128 x 128, laid out [row block][column block]."""

    def __init__(self, data: Tensor, scales: Tensor, tiles: bool):
        _matrix(data, "Fp8Tensor", DType.float8_e4m3)
        _matrix(scales, "Fp8Tensor scales", DType.float32)
        rows, cols = data.shape()
        blocks = -(-cols // BLOCK)
        if scales.shape() != ([-(-rows // BLOCK), blocks] if tiles else [blocks, rows]):
            raise RuntimeError("Fp8Tensor: scales do not match the matrix")
        self.data, self.scales, self.tiles = data, scales, tiles

    def shape(self) -> list[int]:
        return self.data.shape()

    @property
    def stream(self):
        return self.data.stream

    def nbytes(self) -> int:
        return self.data.nbytes() + self.scales.nbytes()

    def dequantize(self, dtype: DType = DType.float32) -> Tensor:
        """codes * scales."""
        code = _code(dtype, "dequantize")
        rows, cols = self.shape()
        out = _like(self.data, [rows, cols], dtype)
        _lib.check(_lib.load().cudeep_b200_dequantize_fp8(_ptr(self.data), _ptr(self.scales), rows, cols,
                                                          BLOCK if self.tiles else 1, _ptr(out), code, out.stream))
        return out


def quantize_fp8(x: Tensor, tiles: bool = False) -> Fp8Tensor:
    """x [rows, cols] (float32 or bfloat16) in blocks of 1 x 128, the form of activations and their gradients, or of
    128 x 128 (`tiles`), the form of weights."""
    _matrix(x, "quantize_fp8")
    code = _code(x.dtype(), "quantize_fp8")
    rows, cols = x.shape()
    if cols == 0:
        raise RuntimeError("quantize_fp8: no columns")
    blocks = -(-cols // BLOCK)
    data = _like(x, [rows, cols], DType.float8_e4m3)
    scales = _like(x, [-(-rows // BLOCK), blocks] if tiles else [blocks, rows], DType.float32)
    _lib.check(_lib.load().cudeep_b200_quantize_fp8(_ptr(x), code, rows, cols, BLOCK if tiles else 1, _ptr(data),
                                                    _ptr(scales), x.stream))
    return Fp8Tensor(data, scales, tiles)


def _operands(rows8: Fp8Tensor, w8: Fp8Tensor, what: str) -> None:
    if not isinstance(rows8, Fp8Tensor) or rows8.tiles:
        raise RuntimeError(f"{what}: rows quantised in blocks of 1 x 128 expected")
    if not isinstance(w8, Fp8Tensor) or not w8.tiles:
        raise RuntimeError(f"{what}: a weight quantised with tiles=True expected")


def linear_fp8(x: Fp8Tensor, weight: Fp8Tensor, bias: Optional[Tensor] = None, activation=None,
               dtype: DType = DType.bfloat16) -> Tensor:
    """act(x @ weight^T + bias) of 8-bit operands; weight is [out_features, in_features], bias float32."""
    _operands(x, weight, "linear_fp8")
    m, k = x.shape()
    n, k2 = weight.shape()
    if k != k2:
        raise RuntimeError("linear_fp8: inner dimensions do not match")
    if bias is not None:
        _dense(bias, "linear_fp8 bias", DType.float32)
        if bias.numel() != n:
            raise RuntimeError("linear_fp8: bias must have out_features elements")
    out = _like(x.data, [m, n], dtype)
    _lib.check(_lib.load().cudeep_b200_linear_forward_fp8(
        _ptr(x.data), _ptr(x.scales), _ptr(weight.data), _ptr(weight.scales), _ptr(bias), _ptr(out),
        _code(dtype, "linear_fp8"), m, n, k, _epilogue_code(activation), out.stream))
    return out


def linear_fp8_backward_data(grad: Fp8Tensor, weight: Fp8Tensor, dtype: DType = DType.bfloat16) -> Tensor:
    """grad @ weight of 8-bit operands: the gradient of linear_fp8's input from the same quantised weight."""
    _operands(grad, weight, "linear_fp8_backward_data")
    m, n = grad.shape()
    n2, k = weight.shape()
    if n != n2:
        raise RuntimeError("linear_fp8_backward_data: inner dimensions do not match")
    out = _like(grad.data, [m, k], dtype)
    _lib.check(_lib.load().cudeep_b200_linear_backward_data_fp8(
        _ptr(grad.data), _ptr(grad.scales), _ptr(weight.data), _ptr(weight.scales), _ptr(out),
        _code(dtype, "linear_fp8_backward_data"), m, n, k, out.stream))
    return out


def linear_backward_saved(grad: Tensor, x: Fp8Tensor, weight: Tensor, z: Optional[Fp8Tensor] = None, activation=None,
                          weight_grad_dtype: DType = DType.bfloat16):
    """(dx, dw, db) of act(x @ weight^T + bias) from x and the pre-activation z kept in 8 bits; grad and weight are
    bfloat16, db is float32.  z is not needed without an activation."""
    _matrix(grad, "linear_backward_saved", DType.bfloat16)
    _matrix(weight, "linear_backward_saved", DType.bfloat16)
    m, n = grad.shape()
    n2, k = weight.shape()
    if not isinstance(x, Fp8Tensor) or x.tiles or x.shape() != [m, k] or n != n2:
        raise RuntimeError("linear_backward_saved: grad [m, n], x [m, k] in blocks of 1 x 128 and weight [n, k] expected")
    act = _epilogue_code(activation)
    if act != 0 and (not isinstance(z, Fp8Tensor) or z.tiles or z.shape() != [m, n]):
        raise RuntimeError("linear_backward_saved: an activation needs z [m, n] in blocks of 1 x 128")
    dx, dw = _like(grad, [m, k], DType.bfloat16), _like(grad, [n, k], weight_grad_dtype)
    db = _like(grad, [n], DType.float32)
    _lib.check(_lib.load().cudeep_b200_linear_backward_saved_fp8(
        _ptr(grad), _code(grad.dtype(), "grad"), _ptr(x.data), _ptr(x.scales), _ptr(z.data) if act else None,
        _ptr(z.scales) if act else None, act, _ptr(weight), _ptr(dx), _ptr(dw),
        _code(weight_grad_dtype, "linear_backward_saved"), _ptr(db), m, n, k, grad.stream))
    return dx, dw, db


def _groups(offsets: Tensor, weight: Tensor, what: str) -> int:
    if not isinstance(offsets, Tensor) or offsets.ndim() != 1:
        raise RuntimeError(f"{what}: offsets is a 1-D Tensor")
    _dense(offsets, what, DType.int32)
    if not isinstance(weight, Tensor) or weight.ndim() != 3:
        raise RuntimeError(f"{what}: weight [groups, out_features, in_features] expected")
    _dense(weight, what, DType.bfloat16)
    groups = offsets.numel() - 1
    if groups < 1 or weight.shape()[0] != groups:
        raise RuntimeError(f"{what}: offsets must have one element more than there are groups")
    return groups


def grouped_linear(x: Tensor, weight: Tensor, offsets: Tensor) -> Tensor:
    """y[r] = x[r] @ weight[g]^T for the rows r in [offsets[g], offsets[g + 1]) of each group g; other rows are zero.
    offsets is an int32 Tensor on the device, so group sizes may come from a kernel."""
    groups = _groups(offsets, weight, "grouped_linear")
    _matrix(x, "grouped_linear", DType.bfloat16)
    rows, k = x.shape()
    n = weight.shape()[1]
    if weight.shape()[2] != k:
        raise RuntimeError("grouped_linear: inner dimensions do not match")
    out = _zeros(x, [rows, n])
    _lib.check(_lib.load().cudeep_b200_grouped_matmul_nt(_ptr(x), _ptr(weight), _ptr(out), 2, _ptr(offsets), groups,
                                                         rows, n, k, x.stream))
    return out


def grouped_linear_backward(grad: Tensor, x: Tensor, weight: Tensor, offsets: Tensor,
                            weight_grad_dtype: DType = DType.float32):
    """(dx, dweight) of grouped_linear; rows of no group get zeros, a group without rows a zero gradient."""
    groups = _groups(offsets, weight, "grouped_linear_backward")
    _matrix(grad, "grouped_linear_backward", DType.bfloat16)
    _matrix(x, "grouped_linear_backward", DType.bfloat16)
    rows, k = x.shape()
    n = weight.shape()[1]
    if weight.shape()[2] != k or grad.shape() != [rows, n]:
        raise RuntimeError("grouped_linear_backward: grad [rows, out_features] and x [rows, in_features] expected")
    dx = _zeros(x, [rows, k])
    dw = _like(x, weight.shape(), weight_grad_dtype)
    lib = _lib.load()
    _lib.check(lib.cudeep_b200_grouped_matmul_nn(_ptr(grad), _ptr(weight), _ptr(dx), 2, _ptr(offsets), groups, rows, k,
                                                 n, x.stream))
    _lib.check(lib.cudeep_b200_grouped_matmul_tn(_ptr(grad), _ptr(x), _ptr(dw), 2,
                                                 _code(weight_grad_dtype, "grouped_linear_backward"), _ptr(offsets),
                                                 groups, rows, n, k, x.stream))
    return dx, dw


def _zeros(ref: Tensor, shape) -> Tensor:
    out = _like(ref, shape, DType.bfloat16)
    # Pairs of bfloat16 zeros are float32 zeros; the pool's blocks are whole multiples of 256 bytes, so an odd last one fits.
    if out.numel():
        _lib.check(_lib.load().cudeep_b200_fill_f32(_ptr(out), 0.0, (out.numel() + 1) // 2, out.stream))
    return out
