"""CPU checks of the scan, dropout and 8-bit product entry points: their
headers are exported, bad arguments are refused before any device work, and the
oracle they are held to agrees with torch's autograd, with differences and with
the published test vectors of its generator."""
import ctypes

import numpy as np
import pytest

from jstorch_b200 import _lib
from oracle import oracle


@pytest.mark.parametrize("header,names", [
    (_lib.SCAN_HEADER, ["jst_scan_backward", "jst_scan_forward"]),
    (_lib.DROPOUT_HEADER, ["jst_dropout"]),
    (_lib.QUANT_HEADER, ["jst_gemm_i8", "jst_linear_i8", "jst_quantize_rows_i8"]),
])
def test_headers_are_exported(header, names):
    assert _lib.header_functions(header) == names
    for n in names:
        assert hasattr(_lib.load(), n)


# addresses far apart that nothing reads: every call below ends on the host
G, H0, LEN, OUT, HN, DOUT, DG, DH0 = (0x10_0000_0000 * (i + 1) for i in range(8))


def _forward(gates=G, ld=16, seq=3, batch=2, hidden=8, h0=H0, lengths=LEN, candidate=0, out=OUT, ld_out=8, h_n=HN):
    return _lib.load().jst_scan_forward(gates, ld, seq, batch, hidden, h0, lengths, 0, candidate, out, ld_out, h_n, None)


@pytest.mark.parametrize("bad", [
    {"seq": -1}, {"batch": -1}, {"hidden": -1}, {"candidate": 2}, {"candidate": -1}, {"ld": 15}, {"ld_out": 7},
    {"gates": None}, {"out": None}, {"out": G}, {"out": G + 4}, {"out": H0}, {"h_n": G + 64}, {"h_n": OUT},
    {"h_n": H0 + 4}, {"ld": 1 << 62}, {"ld_out": 1 << 62},
])
def test_scan_forward_refusals(bad):
    assert _forward(**bad) == 1 and b"scan" in _lib.load().jst_last_error()


def _backward(gates=G, ld=16, seq=3, batch=2, hidden=8, h0=H0, candidate=0, out=OUT, ld_out=8, dout=DOUT, ld_dout=8,
              dh_n=HN, dgates=DG, ld_dg=16, dh0=DH0):
    return _lib.load().jst_scan_backward(gates, ld, seq, batch, hidden, h0, LEN, 0, candidate, out, ld_out, dout,
                                         ld_dout, dh_n, dgates, ld_dg, dh0, None)


@pytest.mark.parametrize("bad", [
    {"seq": -1}, {"candidate": 3}, {"ld": 15}, {"ld_out": 7}, {"ld_dout": 7}, {"ld_dg": 15}, {"gates": None},
    {"out": None}, {"dgates": None}, {"dgates": G}, {"dgates": OUT}, {"dgates": DOUT + 4}, {"dh0": H0}, {"dh0": DG},
    {"dh0": OUT}, {"dh0": HN + 4}, {"ld_dg": 1 << 62}, {"ld_dout": 1 << 62},
])
def test_scan_backward_refusals(bad):
    assert _backward(**bad) == 1 and b"scan" in _lib.load().jst_last_error()


def _dropout(x=G, ldx=8, y=OUT, ldy=8, rows=4, cols=8, p=0.5):
    return _lib.load().jst_dropout(x, ldx, y, ldy, rows, cols, p, 1, 2, None, None)


@pytest.mark.parametrize("bad", [
    {"rows": -1}, {"cols": -1}, {"p": -0.1}, {"p": 1.1}, {"p": float("nan")}, {"x": None}, {"y": None}, {"ldx": 7},
    {"ldy": 7}, {"y": G + 4}, {"y": G, "ldy": 9}, {"rows": 1 << 40, "cols": 1 << 40}, {"ldx": 1 << 62},
])
def test_dropout_refusals(bad):
    assert _dropout(**bad) == 1 and b"dropout" in _lib.load().jst_last_error()


def _desc(**change):
    d = _lib.GemmI8Desc()
    d.M, d.N, d.K = 4, 5, 16
    d.A, d.lda, d.B, d.ldb, d.C, d.ldc = G, 16, OUT, 16, DG, 5
    d.a_scale, d.b_scale, d.bias = H0, HN, DH0
    for k, v in change.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("bad", [
    {"M": -1}, {"N": -1}, {"K": -1}, {"K": 131072, "lda": 131072, "ldb": 131072}, {"lda": 15}, {"ldb": 15}, {"ldc": 4},
    {"A": None}, {"B": None}, {"C": None}, {"a_scale": None}, {"b_scale": None}, {"bias": None, "epilogue": 1},
    {"epilogue": 4}, {"epilogue": 8}, {"epilogue": -1}, {"lda": 1 << 62}, {"ldb": 1 << 62}, {"ldc": 1 << 62},
    {"M": 0x7fff0001}, {"N": 0x7fff0001, "ldc": 0x7fff0001}, {"C": G + 60}, {"C": OUT + 76},
])
def test_gemm_i8_refusals(bad):
    lib = _lib.load()
    assert lib.jst_gemm_i8(ctypes.byref(_desc(**bad))) == 1 and b"gemm_i8" in lib.jst_last_error()
    assert lib.jst_gemm_i8(None) == 1


def _linear(x=G, ldx=16, M=4, K=16, w=OUT, ldw=16, ws=HN, N=5, bias=DH0, epilogue=1, y=DG, ldy=5):
    return _lib.load().jst_linear_i8(x, ldx, M, K, w, ldw, ws, N, bias, epilogue, y, ldy, None)


@pytest.mark.parametrize("bad", [
    {"M": -1}, {"K": 131072, "ldx": 131072, "ldw": 131072}, {"x": None}, {"w": None}, {"ws": None}, {"y": None},
    {"bias": None}, {"epilogue": 5}, {"ldx": 15}, {"ldw": 15}, {"ldy": 4}, {"ldx": 1 << 62},
    {"M": 0x7fff0001}, {"N": 0x7fff0001, "ldy": 0x7fff0001}, {"y": G + 240}, {"y": OUT + 76},
])
def test_linear_i8_refusals(bad):
    assert _linear(**bad) == 1


def test_quantize_rows_refusals():
    lib = _lib.load()
    good = dict(x=G, ldx=16, rows=4, cols=16, q=OUT, ldq=16, scale=HN)
    for bad in ({"rows": -1}, {"cols": -1}, {"x": None}, {"q": None}, {"scale": None}, {"ldx": 15}, {"ldq": 15},
                {"ldx": 1 << 62}, {"ldq": 1 << 62}, {"q": G + 32}, {"scale": G}, {"scale": OUT + 60},
                {"rows": 0x7fff0001}, {"rows": 1, "cols": 0x7fff0001}):
        a = {**good, **bad}
        assert lib.jst_quantize_rows_i8(a["x"], a["ldx"], a["rows"], a["cols"], a["q"], a["ldq"], a["scale"], None) == 1


def test_no_device_is_an_error():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert _forward() == 8 and _backward() == 8 and _dropout() == 8 and _linear() == 8
    assert _lib.load().jst_gemm_i8(ctypes.byref(_desc())) == 8


def test_python_entry_points_refuse_host_tensors():
    import torch

    import jstorch_b200
    from jstorch_b200 import quant, rnn
    x, q = torch.zeros(3, 4), torch.zeros((3, 4), dtype=torch.int8)
    for call in (lambda: jstorch_b200.dropout(x, 0.5, 1), lambda: quant.quantize_rows(x),
                 lambda: quant.linear_i8(x, q, torch.zeros(3)), lambda: quant.gemm_i8(q, q, x[0], x[0]),
                 lambda: rnn.gated_scan(torch.zeros(2, 3, 4))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: jstorch_b200.dropout(x.double(), 0.5, 1), lambda: quant.gemm_i8(x, q, x[0], x[0]),
                 lambda: rnn.gated_scan([1.0])):
        with pytest.raises(TypeError):
            call()


# ------------------------------------------------------------------ the oracle
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("tanh", [False, True])
def test_scan_oracle_against_autograd_and_differences(reverse, tanh):
    import torch
    rng = np.random.default_rng(5)
    seq, batch, hidden, lengths = 9, 4, 3, [9, 0, 1, 6]
    gates, h0 = rng.standard_normal((seq, batch, 2 * hidden)) * 2, rng.standard_normal((batch, hidden))
    dout, dh_n = rng.standard_normal((seq, batch, hidden)), rng.standard_normal((batch, hidden))

    def loss(gates, h0):
        h, total = h0, 0.0
        for t in (range(seq - 1, -1, -1) if reverse else range(seq)):
            z = torch.sigmoid(gates[t, :, :hidden])
            n = gates[t, :, hidden:]
            n = torch.tanh(n) if tanh else n
            k = torch.tensor([[t < length] for length in lengths])
            h = torch.where(k, z * h + (1 - z) * n, h)
            total = total + (h * k * torch.from_numpy(dout[t])).sum()
        return total + (h * torch.from_numpy(dh_n)).sum()

    tg, th = torch.from_numpy(gates).requires_grad_(), torch.from_numpy(h0).requires_grad_()
    loss(tg, th).backward()
    r = oracle.scan_f64(gates, h0, lengths, reverse, tanh, dout, dh_n, with_grads=True)
    np.testing.assert_allclose(r["dgates"][0], tg.grad.numpy(), rtol=0, atol=1e-12)
    np.testing.assert_allclose(r["dh0"][0], th.grad.numpy(), rtol=0, atol=1e-12)

    def value(g, h):
        v = oracle.scan_f64(g, h, lengths, reverse, tanh)
        return float((v["out"][0] * dout).sum() + (v["h_n"][0] * dh_n).sum())

    step = 1e-6  # central differences: off by step^2 times a third derivative of order one, and by 1e-16 / step
    for at in ((0, 0, 1), (5, 0, 4), (3, 3, 2), (0, 2, 5), (7, 3, 0)):
        up, down = gates.copy(), gates.copy()
        up[at] += step
        down[at] -= step
        assert abs((value(up, h0) - value(down, h0)) / (2 * step) - r["dgates"][0][at]) < 1e-8


def test_generator_oracle_against_published_vectors():
    ones = 0xFFFFFFFF
    counters = [[0, 0, 0, 0], [ones] * 4, [0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344]]
    keys = [(0, 0), (ones, ones), (0xA4093822, 0x299F31D0)]
    words = [[0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8], [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD],
             [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]]
    for c, k, w in zip(counters, keys, words):
        assert oracle.philox4x32_10([c], k)[0].tolist() == w


def test_dropout_oracle_keeps_the_right_share():
    n, p = 1 << 20, 0.3
    keep = oracle.dropout_keep(n, p, 7, 9)
    assert abs(keep.mean() - (1 - p)) < 6 * (p * (1 - p) / n) ** 0.5  # six standard deviations
    assert not np.array_equal(keep, oracle.dropout_keep(n, p, 7, 10))
    assert not np.array_equal(keep, oracle.dropout_keep(n, p, 8, 9))


def test_quantize_oracle():
    x = np.array([[127.0, 0.5, 1.5, -2.5, -127.0], [0, 0, 0, 0, 0], [1.0, np.inf, 0, 0, 0], [np.nan, 1, 2, 3, 4]],
                 dtype=np.float32)
    q, s = oracle.quantize_rows(x)
    assert q[0].tolist() == [127, 0, 2, -2, -127] and s[0] == 1.0  # ties to even
    assert not q[1:].any() and s[1] == 0 and np.isnan(s[2:]).all()
