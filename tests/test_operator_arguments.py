"""What the C entry points of the scan, the dropout and the 8-bit products take and refuse, on the host alone."""
import ctypes

import pytest
import torch

from jstorch_b200 import _lib

# addresses far apart that nothing reads: a call that is taken ends at the missing device
G, H0, LEN, OUT, HN, DOUT, DG, DH0 = (0x10_0000_0000 * (i + 1) for i in range(8))
SHARED = 0x10_0000_0000 * 20
TAKEN = 0 if torch.cuda.is_available() else 8  # JST_OK, JST_ERR_NO_DEVICE


def _gemm(**change):
    d = _lib.GemmI8Desc()
    d.M, d.N, d.K = 4, 5, 16
    d.A, d.lda, d.B, d.ldb, d.C, d.ldc = G, 16, OUT, 16, DG, 5
    d.a_scale, d.b_scale, d.bias, d.epilogue = H0, HN, DH0, 1
    for k, v in change.items():
        setattr(d, k, v)
    return _lib.load().jst_gemm_i8(ctypes.byref(d))


def _linear(x=G, ldx=16, M=4, K=16, w=OUT, ldw=16, ws=HN, N=5, bias=DH0, epilogue=1, y=DG, ldy=5):
    return _lib.load().jst_linear_i8(x, ldx, M, K, w, ldw, ws, N, bias, epilogue, y, ldy, None)


@pytest.mark.parametrize("empty", [{"M": 0}, {"N": 0}])
def test_an_empty_product_needs_no_pointer(empty):
    """An empty tensor has no address: neither operands nor the bias of an epilogue."""
    none = dict.fromkeys(("A", "B", "C", "a_scale", "b_scale", "bias"))
    assert _gemm(**empty, **none) == TAKEN
    assert _linear(**empty, x=None, w=None, ws=None, bias=None, y=None) == TAKEN


@pytest.mark.parametrize("vector", ["a_scale", "b_scale", "bias"])
def test_a_product_does_not_overwrite_its_vectors(vector):
    """Blocks read scales and bias while others write C."""
    for at in (DG, DG + 76, DG - 12):  # C is 80 bytes
        assert _gemm(**{vector: at}) == 1 and b"overlaps" in _lib.load().jst_last_error()
    if vector != "a_scale":
        assert _linear(**{"b_scale": {"ws": DG + 76}, "bias": {"bias": DG - 16}}[vector]) == 1
    assert _gemm(bias=DG, epilogue=0, M=0) == TAKEN


def _forward(gates=G, ld=16, seq=3, batch=2, hidden=8, h0=H0, lengths=LEN, out=OUT, ld_out=8, h_n=HN):
    return _lib.load().jst_scan_forward(gates, ld, seq, batch, hidden, h0, lengths, 0, 0, out, ld_out, h_n, None)


def _backward(gates=G, ld=16, seq=3, batch=2, hidden=8, h0=H0, lengths=LEN, out=OUT, ld_out=8, dout=DOUT, ld_dout=8, dh_n=HN,
              dgates=DG, ld_dg=16, dh0=DH0):
    return _lib.load().jst_scan_backward(gates, ld, seq, batch, hidden, h0, lengths, 0, 0, out, ld_out, dout, ld_dout, dh_n,
                                         dgates, ld_dg, dh0, None)


@pytest.mark.parametrize("call,where", [(_forward, (OUT, OUT + 188, OUT - 4, HN, HN + 60)),
                                        (_backward, (DG, DG + 380, DG - 4, DH0, DH0 + 60))])
def test_a_scan_does_not_overwrite_its_lengths(call, where):
    """Every block reads them; blocks of one cluster have to read the same."""
    for at in where:
        assert call(lengths=at) == 1 and b"overlaps" in _lib.load().jst_last_error()


def _dropout(x=G, ldx=8, y=OUT, ldy=8, rows=4, cols=8, p=0.5, step=None):
    return _lib.load().jst_dropout(x, ldx, y, ldy, rows, cols, p, 1, 2, step, None)


def test_dropout_does_not_overwrite_its_step():
    """Every thread reads it."""
    for at in (OUT, OUT + 120, OUT - 4):
        assert _dropout(step=at) == 1 and b"overlaps" in _lib.load().jst_last_error()


def _quantize(x=G, ldx=16, rows=4, cols=16, q=OUT, ldq=16, scale=HN):
    return _lib.load().jst_quantize_rows_i8(x, ldx, rows, cols, q, ldq, scale, None)


@pytest.mark.skipif(TAKEN == 0, reason="calls that are taken run, and these addresses are nobody's")
def test_column_ranges_of_one_matrix_are_no_overlap():
    """Operand and output in the same rows of one buffer, side by side."""
    for call, one, other in (
            (lambda a, b: _forward(gates=a, ld=24, out=b, ld_out=24), 64, 32),
            (lambda a, b: _backward(gates=a, ld=32, dgates=b, ld_dg=32), 64, 64),
            (lambda a, b: _backward(out=a, ld_out=24, dgates=b, ld_dg=24), 32, 64),
            (lambda a, b: _backward(dout=a, ld_dout=24, dgates=b, ld_dg=24), 32, 64),
            (lambda a, b: _dropout(x=a, ldx=16, y=b, ldy=16), 32, 32),
            (lambda a, b: _gemm(A=a, lda=36, C=b, ldc=9), 16, 20),
            (lambda a, b: _gemm(B=a, ldb=36, C=b, ldc=9), 16, 20),
            (lambda a, b: _linear(x=a, ldx=21, y=b, ldy=21), 64, 20),
            (lambda a, b: _quantize(x=a, ldx=20, q=b, ldq=80), 64, 16)):
        for a, b in ((SHARED, SHARED + one), (SHARED + other, SHARED)):
            assert call(a, b) == TAKEN
        for a, b in ((SHARED, SHARED + one - 4), (SHARED + other - 4, SHARED), (SHARED + 4, SHARED)):  # a column in both
            assert call(a, b) == 1 and b"overlap" in _lib.load().jst_last_error()


def test_other_pitches_and_vectors_within_a_matrix_are():
    """Rows of different pitches cross sooner or later; a vector of several rows' length covers what lies between."""
    assert _dropout(x=G, ldx=16, y=G + 32, ldy=17) == 1
    assert _forward(gates=G, ld=24, h_n=G + 64) == 1
    assert _gemm(C=G, ldc=9, a_scale=G + 24) == 1


def test_another_torch_needs_another_build(monkeypatch):
    """The extension is bound to one build of torch: not used with another, and built again for it."""
    from jstorch_b200 import build
    build.build_calls()
    assert _lib.calls().torch_version == torch.__version__
    commands = []
    monkeypatch.setattr(build, "_run", lambda cmd, verbose: commands.append(cmd))
    monkeypatch.setattr(build.os, "replace", lambda a, b: None)
    build.build_calls()
    assert not commands
    monkeypatch.setattr(_lib, "_calls", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    with pytest.raises(ImportError, match="jstorch_b200.build"):
        _lib.calls()
    stamp = build.BUILD / "calls.torch"
    held = stamp.read_text()
    try:
        build.build_calls()
        assert len(commands) == 2 and any("0.0.1" in part for part in commands[0])
    finally:
        stamp.write_text(held)
