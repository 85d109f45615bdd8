"""MXFP4 (microscaled 4-bit floating point) rows and their product, on the GPU.

A block is 32 consecutive values of a row: e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives) under one power-of-two scale, 4.25 bits a value. gfx950's matrix cores multiply
such blocks directly at four times their 16-bit rate.

  quantize(x)              MxTensor of x [rows, k] (float32, bfloat16 or float16)
  dequantize(q, dtype)     the values the codes stand for
  roundtrip(x)             quantize then dequantize, in x's dtype
  matmul(a, b, dtype)      a b^T of two MxTensors
  linear(x, w)             x w^T for MXFP4 weights; x is quantized inside the call

k is a multiple of 32. The exponent of a block is floor(log2 max|x|) - 2; codes round to
nearest even and saturate at 6; a block that holds a NaN or an infinity decodes to NaN.

For inference: the codes carry no gradient, and a backward pass through roundtrip or linear
raises NotImplementedError.
"""
from typing import NamedTuple

import numpy as np
import torch

from . import _lib

BLOCK = 32
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class MxTensor(NamedTuple):
    """MXFP4 rows on the GPU.

    codes: uint8 [rows, k / 2], the even column in the low four bits.
    scales: uint8 [ceil(k / 128), ceil(rows / 64), 4, 16, 4], the exponent (bias 127) of
    row r's block b at [b // 4, r // 64, b % 4, r % 16, r // 16 % 4]: the order the matrix
    cores take them in. Entries of no row or block are not read, except that the blocks
    past the end of a row must not be 255.
    """
    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return (self.codes.shape[0], 2 * self.codes.shape[1])


def scale_shape(rows, k):
    """The shape of an MxTensor's scales."""
    return (-(-k // 128), -(-rows // 64), 4, 16, 4)


def block_scales(q):
    """uint8 [rows, k / 32]: every block's exponent byte, by row (a copy)."""
    rows, k = q.shape
    s = q.scales.permute(1, 4, 3, 0, 2).reshape(-1, 4 * q.scales.shape[0])
    return s[:rows, : k // BLOCK].contiguous()


def _dtype(dt, what):
    code = DTYPES.get(dt)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {dt}")
    return code


def _rows(x):
    """x as [rows, k] whose rows the kernels can read in place: unit column stride, 16-byte
    aligned rows (copied where they are not)."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    step = 16 // x.element_size()
    if x.stride(1) != 1 or x.data_ptr() % 16 or (x.shape[0] > 1 and (
            x.stride(0) % step or x.stride(0) < x.shape[1])):
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _checked(q, what):
    """(rows, k) of an MxTensor whose buffers have the shapes they claim."""
    if not (isinstance(q, tuple) and len(q) == 2):
        raise TypeError(f"{what} must be an MxTensor, got {type(q).__name__}")
    codes, scales = q
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError(f"{what}: codes and scales are uint8")
    if not (codes.is_cuda and scales.is_cuda):
        raise ValueError(f"{what} must be on the GPU")
    if codes.dim() != 2 or not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError(f"{what}: contiguous codes [rows, k / 2] and scales")
    rows, k = codes.shape[0], 2 * codes.shape[1]
    if k == 0 or k % BLOCK or tuple(scales.shape) != scale_shape(rows, k):
        raise ValueError(f"{what}: scales {tuple(scales.shape)} do not fit codes "
                         f"{tuple(codes.shape)}")
    return rows, k


def quantize(x):
    """MxTensor of x [rows, k] (or [..., k], leading dimensions flattened): a CUDA tensor, or
    host data, which is moved to the GPU as float32."""
    lib = _lib.load()
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        x, _ = _lib.to_device(x, torch.float32)
    code = _dtype(x.dtype, "x")
    if x.dim() < 1 or x.shape[-1] == 0 or x.shape[-1] % BLOCK:
        raise ValueError(f"rows of {tuple(x.shape)} do not hold whole blocks of {BLOCK}")
    x = _rows(x)
    rows, k = x.shape
    codes = x.new_empty((rows, k // 2), dtype=torch.uint8)
    scales = x.new_empty(scale_shape(rows, k), dtype=torch.uint8)
    _lib.check(lib.cp_mx4_quantize(x.data_ptr(), code, rows, k, x.stride(0), codes.data_ptr(),
                                   scales.data_ptr(), _lib.stream_ptr()))
    return MxTensor(codes, scales)


def dequantize(q, dtype=torch.float32):
    """[rows, k] of ``dtype``: the codes' values, rounded once (exact in float32)."""
    lib = _lib.load()
    code = _dtype(dtype, "dtype")
    rows, k = _checked(q, "q")
    y = q.codes.new_empty((rows, k), dtype=dtype)
    _lib.check(lib.cp_mx4_dequantize(q.codes.data_ptr(), q.scales.data_ptr(), rows, k,
                                     y.data_ptr(), code, _lib.stream_ptr()))
    return y


def roundtrip(x):
    """x through MXFP4 and back, in its own dtype and shape. Host data comes back as numpy, in
    float32 where it is neither float16 nor float64."""
    if isinstance(x, torch.Tensor) and x.is_cuda:
        y = dequantize(quantize(x), x.dtype).reshape(x.shape)
        return _lib.no_backward(y, "mxfp4.roundtrip", x)
    x = x.detach() if isinstance(x, torch.Tensor) else np.asarray(x)
    y = _lib.to_host(dequantize(quantize(x))).reshape(tuple(x.shape))
    own = str(x.dtype).rpartition(".")[2]
    return y.astype(own) if own in ("float16", "float64") else y


def matmul(a, b, dtype=torch.bfloat16):
    """[m, n] of ``dtype``: a [m, k] times b [n, k]^T, summed in float32, rounded once."""
    lib = _lib.load()
    code = _dtype(dtype, "dtype")
    m, k = _checked(a, "a")
    n, kb = _checked(b, "b")
    if k != kb:
        raise ValueError(f"rows of {k} times rows of {kb}")
    y = a.codes.new_empty((m, n), dtype=dtype)
    nws = lib.cp_mx4_matmul_ws_bytes(m, n, k)
    ws = _lib.workspace(nws, y.device) if nws else None
    _lib.check(lib.cp_mx4_matmul(a.codes.data_ptr(), a.scales.data_ptr(), m, b.codes.data_ptr(),
                                 b.scales.data_ptr(), n, k, y.data_ptr(), code, _lib.ptr(ws), nws,
                                 _lib.stream_ptr()))
    return y


def linear(x, w, dtype=None):
    """x [..., k] times w [n, k]^T -> [..., n] of ``dtype`` (x's by default). x is a CUDA
    tensor and is quantized as quantize() does inside the call; the products of the codes
    are summed in float32 and rounded once."""
    lib = _lib.load()
    xc = _dtype(x.dtype if isinstance(x, torch.Tensor) else type(x).__name__, "x")
    dtype = dtype or x.dtype
    yc = _dtype(dtype, "dtype")
    n, k = _checked(w, "w")
    if not x.is_cuda:
        raise ValueError("x must be on the GPU")
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x {tuple(x.shape)} for weights of {k} columns")
    rows = _rows(x)
    m = rows.shape[0]
    y = x.new_empty(x.shape[:-1] + (n,), dtype=dtype)
    nws = lib.cp_mx4_linear_ws_bytes(m, n, k)
    ws = _lib.workspace(nws, x.device) if nws else None
    _lib.check(lib.cp_mx4_linear(rows.data_ptr(), xc, m, rows.stride(0), w.codes.data_ptr(),
                                 w.scales.data_ptr(), n, k, y.data_ptr(), yc, _lib.ptr(ws), nws,
                                 _lib.stream_ptr()))
    return _lib.no_backward(y, "mxfp4.linear", x)
