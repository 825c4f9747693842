"""8-bit integer matrix products (include/jstorch_quant.h) on torch CUDA tensors:
one scale a token, one scale a channel, exact integer sums.

    q, s = quantize_rows(w)                      # a weight [out, in], once
    y = linear_i8(x, q, s, bias=b)               # fp32 rows in and out
    y = gemm_i8(xq, q, x_scale, s, bias=b)       # rows quantised before
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib


def _matrix(x, name: str):
    """(rows, cols, pitch) of a 2-D tensor whose columns are adjacent."""
    if x.dim() != 2:
        raise ValueError(f"{name} must be 2-D")
    rows, cols = x.shape
    if max(rows, cols) > 0x7fff0000:
        raise ValueError(f"{name}: size > 0x7fff0000")
    if x.is_contiguous():
        return rows, cols, cols or 1
    pitch, unit = x.stride()
    if (cols > 1 and unit != 1) or (rows > 1 and pitch < cols):
        raise ValueError(f"{name}: unsupported strides {tuple(x.stride())} for shape {tuple(x.shape)}")
    return rows, cols, pitch if rows > 1 else max(cols, 1)


def _require_i8(x, name: str) -> int:
    """The device index of x; raises unless x is an int8 CUDA tensor."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if x.dtype is not torch.int8:
        raise TypeError(f"{name} must be int8 (got {x.dtype})")
    index = x.get_device()
    if index < 0 or not x.is_cuda:
        raise ValueError(f"{name} must live on a CUDA device")
    return index


def _vector(v, name: str, n: int, index: int):
    """Address of n adjacent float32 values on device `index`."""
    if _lib.require_f32(v, name) != index or v.shape != (n,) or not v.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor with {n} elements on cuda:{index}")
    return v.data_ptr()


def _output(out, like, M: int, N: int, index: int, stream):
    """(out, its pitch): a float32 [M, N] tensor, made where none is given."""
    if out is None:
        return _lib.empty(like, (M, N), stream), N or 1
    if _lib.require_f32(out, "out") != index or out.shape != (M, N):
        raise ValueError(f"out must be a float32 tensor of shape {(M, N)} on cuda:{index}")
    return out, _matrix(out, "out")[2]


def quantize_rows(x, *, stream=None):
    """(q, scale) of a 2-D float32 CUDA tensor: scale[r] = max|x[r]| * (1 / 127)
    in fp32, q[r] = x[r] / scale[r] to the nearest integer (ties to even) in int8.
    A row that holds an infinity or a NaN gets scale NaN.  The rows of q start
    at multiples of 16 bytes (q is a view when x has other widths), as
    gemm_i8 reads them in place.
    """
    index = _lib.require_f32(x, "x")
    rows, cols, ldx = _matrix(x, "x")
    pitch = max((cols + 15) // 16 * 16, 16)
    scale = _lib.empty(x, (rows,), stream)
    held = _lib.empty(x, (rows, pitch // 4), stream).view(torch.int8)
    _lib.call(index, stream, _lib.load().jst_quantize_rows_i8, x.data_ptr(), ldx, rows, cols, held.data_ptr(), pitch,
              scale.data_ptr())
    return held[:, :cols], scale


def _run_desc(d, handle) -> int:
    d.stream = handle
    return _lib.load().jst_gemm_i8(ctypes.byref(d))


def gemm_i8(a, w, a_scale, w_scale, out=None, *, bias=None, relu: bool = False, stream=None):
    """out[m, n] = relu?(a_scale[m] * w_scale[n] * sum_k a[m, k] * w[n, k] + bias[n]).

    a: [M, K] int8 rows (tokens), w: [N, K] int8 rows (channels, an nn.Linear
    weight); K <= 131071.  Rows may have a pitch; 16-byte aligned rows are read
    in place, others are copied first where the tensor cores compute.  out:
    float32 [M, N] (a pitch is allowed).  Runs asynchronously on `stream`
    (default: torch's current stream).
    """
    index = _require_i8(a, "a")
    if _require_i8(w, "w") != index:
        raise ValueError("a and w must live on one device")
    M, K, lda = _matrix(a, "a")
    N, Kw, ldw = _matrix(w, "w")
    if K != Kw:
        raise ValueError(f"gemm_i8 shape mismatch: a is [{M}, {K}], w is [{N}, {Kw}]")
    d = _lib.GemmI8Desc(M, N, K, a.data_ptr(), lda, w.data_ptr(), ldw, _vector(a_scale, "a_scale", M, index),
                        _vector(w_scale, "w_scale", N, index), _vector(bias, "bias", N, index) if bias is not None else None,
                        (_lib.EPI_BIAS if bias is not None else 0) | (_lib.EPI_RELU if relu else 0))
    out, d.ldc = _output(out, a_scale, M, N, index, stream)
    d.C = out.data_ptr()
    _lib.call(index, stream, _run_desc, d)
    return out


def linear_i8(x, w, w_scale, out=None, *, bias=None, relu: bool = False, stream=None):
    """gemm_i8 of quantize_rows(x): x [M, K] float32 rows (a pitch is allowed),
    w [N, K] int8 with w_scale [N] (quantize_rows of the weight), out float32
    [M, N].  The same result as the two calls, in fewer passes.
    """
    index = _lib.require_f32(x, "x")
    if _require_i8(w, "w") != index:
        raise ValueError("x and w must live on one device")
    M, K, ldx = _matrix(x, "x")
    N, Kw, ldw = _matrix(w, "w")
    if K != Kw:
        raise ValueError(f"linear_i8 shape mismatch: x is [{M}, {K}], w is [{N}, {Kw}]")
    scale = _vector(w_scale, "w_scale", N, index)
    b = _vector(bias, "bias", N, index) if bias is not None else None
    out, ldy = _output(out, x, M, N, index, stream)
    _lib.call(index, stream, _lib.load().jst_linear_i8, x.data_ptr(), ldx, M, K, w.data_ptr(), ldw, scale, N, b,
              (_lib.EPI_BIAS if bias is not None else 0) | (_lib.EPI_RELU if relu else 0), out.data_ptr(), ldy)
    return out
