"""8-bit integer matrix products (include/jstorch_quant.h) on torch CUDA tensors:
one scale a token, one scale a channel, exact integer sums.

    q, s = quantize_rows(w)                      # a weight [out, in], once
    y = linear_i8(x, q, s, bias=b)               # fp32 rows in and out
    y = gemm_i8(xq, q, x_scale, s, bias=b)       # rows quantised before
"""
from __future__ import annotations

from . import _lib


def quantize_rows(x, *, stream=None):
    """(q, scale) of a 2-D float32 CUDA tensor: scale[r] = max|x[r]| / 127
    rounded to fp32, q[r] = x[r] / scale[r] to the nearest integer (ties to even) in int8.
    A row that holds an infinity or a NaN gets scale NaN.  The rows of q start
    at multiples of 16 bytes (q is a view when x has other widths), as
    gemm_i8 reads them in place.
    """
    return _lib.calls().quantize_rows(x, stream)


def gemm_i8(a, w, a_scale, w_scale, out=None, *, bias=None, relu: bool = False, stream=None):
    """out[m, n] = relu?(a_scale[m] * w_scale[n] * sum_k a[m, k] * w[n, k] + bias[n]).

    a: [M, K] int8 rows (tokens), w: [N, K] int8 rows (channels, an nn.Linear
    weight); K <= 131071.  Rows may have a pitch; 16-byte aligned rows are read
    in place, others are copied first where the tensor cores compute.  out:
    float32 [M, N] (a pitch is allowed).  Runs asynchronously on `stream`
    (default: torch's current stream).
    """
    return _lib.calls().gemm_i8(a, w, a_scale, w_scale, out, bias, relu, stream)


def linear_i8(x, w, w_scale, out=None, *, bias=None, relu: bool = False, stream=None):
    """gemm_i8 of quantize_rows(x): x [M, K] float32 rows (a pitch is allowed),
    w [N, K] int8 with w_scale [N] (quantize_rows of the weight), out float32
    [M, N].  The same result as the two calls, in fewer passes.
    """
    return _lib.calls().linear_i8(x, w, w_scale, out, bias, relu, stream)
