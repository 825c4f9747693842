"""gated_scan and gated_scan_backward against the step-by-step fp64 recurrence
of oracle.scan_f64, whose elementwise bounds carry the rounding errors of fp32
arithmetic through the recurrence (derived there)."""
import numpy as np
import pytest

from oracle import oracle

pytestmark = pytest.mark.gpu


def _case(seq, batch, hidden, h0=True, lengths=None, seed=0, spread=2.0):
    rng = np.random.default_rng([seed, seq, batch, hidden])
    gates = rng.standard_normal((seq, batch, 2 * hidden)).astype(np.float32)
    gates[..., :hidden] += (spread * rng.standard_normal(hidden)).astype(np.float32)
    state = lambda: rng.standard_normal((batch, hidden)).astype(np.float32)  # noqa: E731
    return {"gates": gates, "h0": state() if h0 else None, "dh_n": state(),
            "dout": rng.standard_normal((seq, batch, hidden)).astype(np.float32),
            "lengths": None if lengths is None else np.asarray(lengths, dtype=np.int32)}


def _dev(x):
    import torch
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _held(name, got, want):
    value, bound = want
    got = got.cpu().numpy().astype(np.float64)
    assert got.shape == value.shape
    off = np.abs(got - value)
    assert np.all(off <= bound), (name, float(np.max(off - bound)), np.unravel_index(np.argmax(off - bound), off.shape))


def _check(c, reverse, tanh):
    import torch
    from jstorch_b200 import rnn
    how = {"lengths": _dev(c["lengths"]), "reverse": reverse, "candidate": "tanh" if tanh else "identity"}
    gates, h0 = _dev(c["gates"]), _dev(c["h0"])
    out, h_n = rnn.gated_scan(gates, h0, **how)
    dgates, dh0 = rnn.gated_scan_backward(gates, out, _dev(c["dout"]), h0, dh_n=_dev(c["dh_n"]), **how)
    torch.cuda.synchronize()
    want = oracle.scan_f64(c["gates"], c["h0"], c["lengths"], reverse, tanh, c["dout"], c["dh_n"], with_grads=True)
    _held("out", out, want["out"])
    _held("h_n", h_n, want["h_n"])
    _held("dgates", dgates, want["dgates"])
    if c["h0"] is not None:
        _held("dh0", dh0, want["dh0"])
    else:
        assert dh0 is None


SIZES = [(1, 1, 1), (1, 3, 5), (2, 1, 32), (7, 2, 31), (8, 1, 33), (9, 5, 64), (31, 1, 8), (63, 3, 10), (64, 2, 96),
         (65, 1, 130), (127, 4, 3), (255, 1, 32), (256, 1, 36), (257, 2, 7), (1000, 1, 40), (1025, 1, 64), (2049, 2, 4),
         (4100, 1, 12), (16, 64, 160), (18, 2200, 64), (33, 300, 130), (40, 400, 51), (70, 80, 128), (300, 40, 64),
         (17, 1, 2), (130, 3, 33)]


@pytest.mark.parametrize("seq,batch,hidden", SIZES)
@pytest.mark.parametrize("reverse,tanh", [(False, True), (True, False)])
def test_sizes(seq, batch, hidden, reverse, tanh):
    _check(_case(seq, batch, hidden, h0=hidden % 2 == 0), reverse, tanh)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("lengths", [[0, 0, 0], [70, 0, 1], [69, 70, 33], [-5, 1000, 64]])
def test_lengths(lengths, reverse):
    _check(_case(70, 3, 20, lengths=lengths), reverse, True)


@pytest.mark.parametrize("reverse", [False, True])
def test_lengths_of_a_long_sequence(reverse):
    _check(_case(3000, 4, 36, lengths=[3000, 1, 0, 1700]), reverse, False)


@pytest.mark.parametrize("reverse", [False, True])
def test_what_lies_behind_a_sequence_does_not_matter(reverse):
    import torch
    from jstorch_b200 import rnn
    lengths = [40, 0, 13, 1]
    c = _case(40, 4, 24, lengths=lengths)
    dirty = {k: None if v is None else v.copy() for k, v in c.items()}
    for b, n in enumerate(lengths):
        dirty["gates"][n:, b] = np.resize(np.array([np.nan, np.inf, -np.inf, 3.4e38], np.float32), (40 - n, 48))
        dirty["dout"][n:, b] = np.nan
    results = []
    for x in (c, dirty):
        g, h0, ln = _dev(x["gates"]), _dev(x["h0"]), _dev(x["lengths"])
        out, h_n = rnn.gated_scan(g, h0, lengths=ln, reverse=reverse)
        back = rnn.gated_scan_backward(g, out, _dev(x["dout"]), h0, dh_n=_dev(x["dh_n"]), lengths=ln, reverse=reverse)
        results.append([t.clone() for t in (out, h_n, *back)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert torch.equal(results[0][1][1], _dev(c["h0"])[1])  # no step: the state passes


def test_extreme_gates():
    """Gates that saturate, zeros, denormals and the largest numbers."""
    import torch
    from jstorch_b200 import rnn
    values = np.array([0.0, -0.0, 1e-40, -1e-40, 87.0, -87.0, 104.0, -104.0, 3.4e38, -3.4e38, np.inf, -np.inf], np.float32)
    n = len(values)
    gates = np.zeros((3, n, 2 * n), np.float32)
    gates[..., :n] = values[None, :, None]  # every a with every c
    gates[..., n:] = values[None, None, :]
    h0 = np.ones((n, n), np.float32)
    out, _ = rnn.gated_scan(_dev(gates), _dev(h0))
    assert not torch.isnan(out).any() and out.abs().max() <= 1.0
    want = oracle.scan_f64(gates, h0, tanh=True)["out"]
    _held("out", out, want)
    # an infinite candidate or a NaN shows in its own channel from its step on, and nowhere else
    g = np.zeros((300, 2, 2 * 40), np.float32)
    g[100, 0, 40 + 3] = np.inf
    g[200, 1, 7] = np.nan
    out, h_n = rnn.gated_scan(_dev(g), None, candidate="identity")
    out = out.cpu().numpy()
    assert np.isposinf(out[100:, 0, 3]).all() and np.isnan(out[200:, 1, 7]).all()
    out[100:, 0, 3] = out[200:, 1, 7] = 0.0
    assert not out.any()


def test_an_infinite_state_stays_infinite():
    """z = 1 / 11 for thousands of steps: products of z underflow, the state does not change."""
    import torch
    from jstorch_b200 import rnn
    for seq in (5, 60, 3000):
        g = torch.zeros((seq, 2, 2 * 40), device="cuda")
        g[..., :40] = -float(np.log(10.0))
        h0 = torch.full((2, 40), float("inf"), device="cuda")
        h0[1] = 1.0
        out, h_n = rnn.gated_scan(g, h0)
        assert bool(torch.isposinf(out[:, 0]).all()) and bool(torch.isposinf(h_n[0]).all())
        assert bool(torch.isfinite(out[:, 1]).all())
        _, dh0 = rnn.gated_scan_backward(torch.zeros_like(g), torch.zeros_like(out), None, torch.zeros_like(h0), dh_n=h0)
        assert bool(torch.isposinf(dh0[0]).all()) and bool(torch.isfinite(dh0[1]).all())


def test_pitches_and_optional_arguments():
    import torch
    from jstorch_b200 import rnn
    seq, batch, hidden = 37, 3, 21
    c = _case(seq, batch, hidden)
    want = oracle.scan_f64(c["gates"], c["h0"], None, False, True, c["dout"], c["dh_n"], with_grads=True)
    wide = torch.full((seq, batch, 2 * hidden + 5), 7.0, device="cuda")
    gates = wide[..., 2:2 + 2 * hidden]
    gates.copy_(_dev(c["gates"]))
    both = torch.full((seq, batch, 2 * hidden + 1), 7.0, device="cuda")
    out = both[..., hidden:2 * hidden]
    h = _dev(c["h0"])
    got, h_n = rnn.gated_scan(gates, h, out=out, h_n=h)  # the state in place
    assert got.data_ptr() == out.data_ptr() and h_n is h
    _held("out", out, want["out"])
    _held("h_n", h_n, want["h_n"])
    assert bool((both[..., :hidden] == 7).all()) and bool((both[..., 2 * hidden:] == 7).all())
    dwide = torch.full((seq, batch, 2 * hidden + 3), 7.0, device="cuda")
    ddout = torch.zeros((seq, batch, hidden + 2), device="cuda")
    ddout[..., 1:1 + hidden].copy_(_dev(c["dout"]))
    dgates, dh0 = rnn.gated_scan_backward(gates, out, ddout[..., 1:1 + hidden], _dev(c["h0"]), dh_n=_dev(c["dh_n"]),
                                          dgates=dwide[..., 1:1 + 2 * hidden])
    _held("dgates", dgates, want["dgates"])
    _held("dh0", dh0, want["dh0"])
    assert bool((dwide[..., 0] == 7).all()) and bool((dwide[..., 1 + 2 * hidden:] == 7).all())
    for dout, dh_n in ((None, c["dh_n"]), (c["dout"], None), (None, None)):
        want = oracle.scan_f64(c["gates"], c["h0"], None, False, True, dout, dh_n, with_grads=True)
        dgates, dh0 = rnn.gated_scan_backward(gates, out, _dev(dout), _dev(c["h0"]), dh_n=_dev(dh_n))
        _held("dgates", dgates, want["dgates"])
        _held("dh0", dh0, want["dh0"])


@pytest.mark.parametrize("seq,batch,hidden", [(0, 3, 8), (5, 0, 8), (5, 3, 0)])
def test_empty(seq, batch, hidden):
    import torch
    from jstorch_b200 import rnn
    gates = torch.zeros((seq, batch, 2 * hidden), device="cuda")
    h0, dh_n = torch.randn((batch, hidden), device="cuda"), torch.randn((batch, hidden), device="cuda")
    out, h_n = rnn.gated_scan(gates, h0)
    dgates, dh0 = rnn.gated_scan_backward(gates, out, torch.zeros_like(out), h0, dh_n=dh_n)
    assert out.shape == (seq, batch, hidden) and dgates.shape == gates.shape
    assert torch.equal(h_n, h0) and torch.equal(dh0, dh_n)
    out, h_n = rnn.gated_scan(gates)
    assert not h_n.any()


def test_repeats_bit_for_bit_in_parts_and_whole():
    """Two calls agree in every bit; a sequence run in two calls that hand the
    state on stays within the bound of one."""
    import torch
    from jstorch_b200 import rnn
    c = _case(1500, 2, 70)
    gates, h0 = _dev(c["gates"]), _dev(c["h0"])
    first, again = rnn.gated_scan(gates, h0), rnn.gated_scan(gates, h0)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    want = oracle.scan_f64(c["gates"], c["h0"])
    a, h = rnn.gated_scan(gates[:611], h0)
    b, h_n = rnn.gated_scan(gates[611:], h)
    _held("out", torch.cat([a, b]), want["out"])
    _held("h_n", h_n, want["h_n"])
    back = [rnn.gated_scan_backward(gates, first[0], _dev(c["dout"]), h0, dh_n=_dev(c["dh_n"])) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*back))


def test_offsets_past_32_bits():
    """More than 2^31 gate values in one call: the last rows are right."""
    import torch
    from jstorch_b200 import rnn
    seq, batch, hidden = 1_050_000, 1, 1024  # 2.15e9 gate values, 1.08e9 outputs
    gates = torch.zeros((seq, batch, 2 * hidden), device="cuda")
    c = _case(64, batch, hidden)
    gates[-64:].copy_(_dev(c["gates"]))
    gates[:-64, :, hidden:] = 0.5  # z = 1/2, n = 1/2: the state settles at 1/2 exactly
    out, h_n = rnn.gated_scan(gates, None, candidate="identity")
    assert bool((out[100:-64] == 0.5).all())
    want = oracle.scan_f64(c["gates"], np.full((batch, hidden), 0.5, np.float32), tanh=False)
    _held("out", out[-64:], want["out"])
    _held("h_n", h_n, want["h_n"])


def test_another_stream_and_a_captured_graph():
    import torch
    from jstorch_b200 import rnn
    c = _case(300, 2, 48)
    gates, h0, dout, dh_n = (_dev(c[k]) for k in ("gates", "h0", "dout", "dh_n"))
    out, h_n = rnn.gated_scan(gates, h0)
    want = [out, h_n, *rnn.gated_scan_backward(gates, out, dout, h0, dh_n=dh_n)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    a, b = rnn.gated_scan(gates, h0, stream=side)
    got = [a, b, *rnn.gated_scan_backward(gates, a, dout, h0, dh_n=dh_n, stream=side)]
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    g = torch.cuda.CUDAGraph()
    held = torch.zeros_like(gates)
    with torch.cuda.graph(g):
        a, b = rnn.gated_scan(held, h0)
        got = [a, b, *rnn.gated_scan_backward(held, a, dout, h0, dh_n=dh_n)]
    for _ in range(2):
        held.copy_(gates)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        held.zero_()


def test_refusals():
    import torch
    from jstorch_b200 import rnn
    g = torch.zeros((4, 2, 12), device="cuda")
    h = torch.zeros((2, 6), device="cuda")
    out = torch.zeros((4, 2, 6), device="cuda")
    bad = [
        lambda: rnn.gated_scan(g[..., :11]), lambda: rnn.gated_scan(g[0]), lambda: rnn.gated_scan(g.transpose(0, 1)),
        lambda: rnn.gated_scan(g.transpose(0, 2)), lambda: rnn.gated_scan(g, h[:1]),
        lambda: rnn.gated_scan(g, torch.zeros((6, 2), device="cuda").t()), lambda: rnn.gated_scan(g, h.cpu()),
        lambda: rnn.gated_scan(g, candidate="relu"), lambda: rnn.gated_scan(g, out=out[:, :, :5]),
        lambda: rnn.gated_scan(g, lengths=torch.zeros(2, device="cuda", dtype=torch.int64)),
        lambda: rnn.gated_scan(g, lengths=torch.zeros(3, device="cuda", dtype=torch.int32)),
        lambda: rnn.gated_scan(g, lengths=torch.zeros(2, dtype=torch.int32)),
        lambda: rnn.gated_scan_backward(g, out[:2], out), lambda: rnn.gated_scan_backward(g, out, out[..., :5]),
        lambda: rnn.gated_scan_backward(g, out, out, dh_n=h[:1]), lambda: rnn.gated_scan_backward(g, out, out, dgates=out),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    from jstorch_b200 import JstError
    for call in (lambda: rnn.gated_scan(g, out=g[..., :6]), lambda: rnn.gated_scan(g, h, h_n=out[0]  , out=out),
                 lambda: rnn.gated_scan_backward(g, out, out, dgates=g)):
        with pytest.raises(JstError, match="overlap"):
            call()


def test_sizes_past_32_bits_are_refused():
    """The C entry points count rows in 32 bits: a larger tensor must not wrap to a smaller one."""
    import torch
    from jstorch_b200 import rnn
    rows = torch.zeros((2 ** 32 + 4, 0), device="cuda")
    for call in (lambda: rnn.gated_scan(rows[:, None]), lambda: rnn.gated_scan(rows[None])):
        with pytest.raises(ValueError, match="size >"):
            call()
