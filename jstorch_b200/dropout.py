"""Dropout through jst_dropout (include/jstorch_dropout.h) on torch CUDA tensors.

The mask is a function of (seed, offset, element index) and is never stored:
the gradient of y = dropout(x, p, seed, offset) is dropout(dy, p, seed, offset).
"""
from __future__ import annotations

from . import _lib


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
    return _lib.calls().dropout(x, p, seed, offset, step, out, stream)
