"""The scan, the dropout and the 8-bit products on views: operands and outputs that share a buffer."""
import numpy as np
import pytest

from oracle import oracle

pytestmark = pytest.mark.gpu


def _held(got, want):
    value, bound = want
    assert np.all(np.abs(got.cpu().numpy().astype(np.float64) - value) <= bound)


@pytest.mark.parametrize("gap", [0, 1])
def test_operands_and_outputs_side_by_side_in_one_buffer(gap):
    """Column ranges of one matrix: results are right and the columns between stay."""
    import torch

    import jstorch_b200
    from jstorch_b200 import quant, rnn
    rng = np.random.default_rng(gap)
    seq, batch, hidden = 70, 3, 26
    g, h0, d = (rng.standard_normal(s).astype(np.float32) for s in ((seq, batch, 52), (batch, 26), (seq, batch, 26)))
    buf = torch.full((seq, batch, 52 + 26 + 26 + 52 + 4 * gap), 7.0, device="cuda")
    at, views = 0, []
    for cols in (52, 26, 26, 52):
        views.append(buf[..., at:at + cols])
        at += cols + gap
    gates, out, dout, dgates = views
    gates.copy_(torch.from_numpy(g))
    dout.copy_(torch.from_numpy(d))
    state = torch.from_numpy(h0).cuda()
    rnn.gated_scan(gates, state, out=out)
    _, dh0 = rnn.gated_scan_backward(gates, out, dout, state, dgates=dgates)
    want = oracle.scan_f64(g, h0, dout=d, with_grads=True)
    for name, got in (("out", out), ("dgates", dgates), ("dh0", dh0)):
        _held(got, want[name])
    assert gap == 0 or bool((buf[..., 52] == 7).all())

    for M in (1, 6, 40, 300):
        K, N = 48, 36
        x = rng.standard_normal((M, K)).astype(np.float32)
        w = rng.integers(-127, 128, (N, K), dtype=np.int8)
        s = rng.uniform(0.5, 1, N).astype(np.float32)
        buf = torch.full((M, K + N + 2 * gap), 7.0, device="cuda")
        buf[:, gap:gap + K] = torch.from_numpy(x)
        y = buf[:, 2 * gap + K:]
        quant.linear_i8(buf[:, gap:gap + K], torch.from_numpy(w).cuda(), torch.from_numpy(s).cuda(), out=y)
        q, xs = oracle.quantize_rows(x)
        _held(y, oracle.gemm_i8_f64(q, w, xs, s))
        assert np.array_equal(buf[:, gap:gap + K].cpu().numpy(), x)
        jstorch_b200.dropout(buf[:, gap:gap + N], 0.5, 3, out=y)
        assert np.array_equal(y.cpu().numpy(), oracle.dropout_f32(x[:, :N], 0.5, 3))


def test_a_negated_view_is_refused():
    """The memory behind the imaginary part of a conjugate holds the negatives of its values."""
    import torch

    import jstorch_b200
    from jstorch_b200 import quant, rnn
    x = torch.randn((6, 1), dtype=torch.complex64, device="cuda").conj().imag
    assert x.is_neg()
    w, one = torch.ones((1, 1), dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda")
    gates = torch.randn((6, 2, 2), dtype=torch.complex64, device="cuda").conj().imag
    out = torch.zeros((6, 1), device="cuda")
    for call in (lambda: quant.quantize_rows(x), lambda: quant.linear_i8(x, w, one), lambda: jstorch_b200.dropout(x, 0.5, 1),
                 lambda: jstorch_b200.dropout(out, 0.5, 1, out=x), lambda: rnn.gated_scan(gates),
                 lambda: quant.linear_i8(out, w, one, bias=x[0])):
        with pytest.raises(ValueError, match="negated"):
            call()
    y = x.resolve_neg()
    assert bool(((quant.linear_i8(x.resolve_neg(), w, one) - y).abs() <= 1e-6 * y.abs()).all())
