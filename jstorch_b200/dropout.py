"""Dropout through jst_dropout (include/jstorch_dropout.h) on torch CUDA tensors.

The mask is a function of (seed, offset, element index) and is never stored:
the gradient of y = dropout(x, p, seed, offset) is dropout(dy, p, seed, offset).
"""
from __future__ import annotations

from . import _lib


def _rows(x, name: str):
    """(rows, cols, pitch) of x as a row-major matrix; contiguous tensors are one row."""
    if x.is_contiguous():
        n = x.numel()
        return 1, n, n
    shape, stride = x.shape, x.stride()
    cols = shape[-1]
    if cols > 1 and stride[-1] != 1:
        raise ValueError(f"{name}: unsupported strides {tuple(stride)} for shape {tuple(shape)}")
    pitch, rows = 0, 1
    for n, st in zip(reversed(shape[:-1]), reversed(stride[:-1])):
        if n == 1:
            continue
        if pitch == 0:
            pitch = st
        if st != pitch * rows or pitch < cols:
            raise ValueError(f"{name}: unsupported strides {tuple(stride)} for shape {tuple(shape)}")
        rows *= n
    return rows, cols, pitch or cols


def dropout(x, p: float, seed: int, offset: int = 0, *, step=None, out=None, stream=None):
    """y = x / (1 - p) where the element is kept (probability 1 - p), else 0.

    x: a float32 CUDA tensor, contiguous or with one pitch between its rows
    (other strides are rejected).  Element i in row-major order draws word
    i % 4 of Philox4x32-10 with counter (i // 4, offset) and key seed (both 64
    bits): give every call under a seed an offset of its own, and the same
    (seed, offset) to forward and backward.  step, a one-element int64 tensor
    on x's device, is added to offset when the kernel runs, so a captured graph
    that advances it draws a new mask at every replay.  out may be x itself.
    Runs asynchronously on `stream` (default: torch's current stream).
    """
    index = _lib.require_f32(x, "x")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1] (got {p})")
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError("seed and offset must be 64-bit unsigned integers")
    if step is not None:
        import torch

        if step.dtype is not torch.int64 or step.numel() != 1 or step.get_device() != index:
            raise ValueError("step must be a one-element int64 tensor on x's device")
        step = step.data_ptr()
    if out is None:
        out = _lib.empty(x, x.shape, stream)
    elif _lib.require_f32(out, "out") != index or out.shape != x.shape:
        raise ValueError(f"out must be a float32 tensor of shape {tuple(x.shape)} on x's device")
    rows, cols, ldx = _rows(x, "x")
    rows_o, cols_o, ldy = _rows(out, "out")
    if (rows, cols) != (rows_o, cols_o):  # one of the two has gaps: the other has rows of the same length without any
        rows, cols = max((rows, cols), (rows_o, cols_o))
        ldx = cols if x.is_contiguous() else ldx
        ldy = cols if out.is_contiguous() else ldy
    _lib.call(index, stream, _lib.load().jst_dropout, x.data_ptr(), ldx, out.data_ptr(), ldy, rows, cols, p, seed, offset,
              step)
    return out
