"""gated_scan and gated_scan_backward where a number meets an edge of its type, and
with lengths in every form of the kernels, against oracle.scan_f64 (bounds derived there)."""
import numpy as np
import pytest

from oracle import oracle

pytestmark = pytest.mark.gpu


def _dev(x):
    import torch
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _held(name, got, want):
    value, bound = want
    got = got.cpu().numpy().astype(np.float64)
    assert got.shape == value.shape
    off = np.abs(got - value)
    assert np.all(off <= bound), (name, float(np.max(off - bound)), np.unravel_index(np.argmax(off - bound), off.shape))


def _check(gates, h0, dout, dh_n, reverse=False, tanh=False, lengths=None):
    from jstorch_b200 import rnn
    how = {"reverse": reverse, "candidate": "tanh" if tanh else "identity", "lengths": _dev(lengths)}
    out, h_n = rnn.gated_scan(_dev(gates), _dev(h0), **how)
    dgates, dh0 = rnn.gated_scan_backward(_dev(gates), out, _dev(dout), _dev(h0), dh_n=_dev(dh_n), **how)
    want = oracle.scan_f64(gates, h0, lengths, reverse, tanh, dout, dh_n, with_grads=True)
    for name, got in (("out", out), ("h_n", h_n), ("dgates", dgates), ("dh0", dh0)):
        _held(name, got, want[name])
    return out, h_n, dgates, dh0


# one lane walks the axis; one block; one and two channels a lane; clusters
FORMS = [(3, 2, 40), (12, 2, 600), (60, 2, 40), (60, 4, 600), (900, 2, 40), (900, 3, 500), (60, 20, 1900)]


@pytest.mark.parametrize("seq,batch,hidden", FORMS)
@pytest.mark.parametrize("a", [-200.0, -np.inf])
def test_a_closed_gate_keeps_nothing(seq, batch, hidden, a):
    """z is 0 there: a state of any size, and a gradient of any size, ends at the step."""
    h0 = np.resize(np.array([1e32, 1e38, -3e38, 1.0], np.float32), (batch, hidden))
    gates = np.zeros((seq, batch, 2 * hidden), np.float32)
    at = np.resize(np.array([0, seq // 2, seq - 1, seq // 3, 1]), hidden)
    gates[at, :, np.arange(hidden)] = a
    gates[..., :hidden][gates[..., :hidden] == 0] = 8.0
    out, h_n, _, dh0 = _check(gates, h0, np.zeros((seq, batch, hidden), np.float32), h0)
    assert not h_n.any() and not dh0.any()
    assert not out.cpu().numpy()[at, :, np.arange(hidden)].any()


@pytest.mark.parametrize("seq,batch,hidden", FORMS)
@pytest.mark.parametrize("reverse", [False, True])
def test_gates_below_the_normal_numbers(seq, batch, hidden, reverse):
    """z or 1 - z around and below 2^-126, next to states of up to 1e38 and candidates of 1e30."""
    rng = np.random.default_rng([seq, hidden])
    gates = rng.standard_normal((seq, batch, 2 * hidden)).astype(np.float32)
    gates[..., hidden:] *= np.float32(1e30)
    edge = rng.random((seq, batch, hidden)) < 0.3
    gates[..., :hidden][edge] = (rng.choice([-1.0, 1.0], edge.sum()) * rng.uniform(80, 108, edge.sum())).astype(np.float32)
    h0, dh_n = (rng.uniform(-1e38, 1e38, (batch, hidden)).astype(np.float32) for _ in range(2))
    # gradients of 1: theirs times the states' 1e38 stays a number
    _check(gates, h0, rng.uniform(-1, 1, (seq, batch, hidden)).astype(np.float32), dh_n * np.float32(1e-38), reverse)


def test_an_infinite_state_and_a_closed_gate():
    """As in arithmetic step by step: infinity times a positive z stays, times 0 is NaN."""
    import torch
    from jstorch_b200 import rnn
    for seq, hidden in ((3, 40), (60, 40), (60, 1300), (3000, 40)):
        for a, kept in ((-80.0, True), (-float("inf"), False)):
            g = torch.zeros((seq, 1, 2 * hidden), device="cuda")
            g[seq // 2, :, :hidden] = a
            h0 = torch.full((1, hidden), float("inf"), device="cuda")
            out, h_n = rnn.gated_scan(g, h0)
            assert bool(torch.isposinf(out[:seq // 2]).all())
            assert bool((torch.isposinf(h_n) if kept else torch.isnan(h_n)).all()), (seq, hidden, a)


@pytest.mark.parametrize("seq,batch,hidden", FORMS)
def test_gradients_where_tanh_saturates(seq, batch, hidden):
    """dn/dc of |c| = 0.5 to 45 keeps its digits (1 - n^2 in fp32 is off by 6 % at 8 and 0 from
    9 on), as far as it is a normal number (to 43.6); at 30 it is 4 e^-60 = 4e-26."""
    rng = np.random.default_rng([seq, hidden, 3])
    gates = rng.standard_normal((seq, batch, 2 * hidden)).astype(np.float32)
    gates[..., hidden:] = rng.choice([-1.0, 1.0], (seq, batch, hidden)) * rng.uniform(0.5, 45, (seq, batch, hidden))
    h0, dh_n = (rng.standard_normal((batch, hidden)).astype(np.float32) for _ in range(2))
    _, _, dgates, _ = _check(gates, h0, rng.standard_normal((seq, batch, hidden)).astype(np.float32), dh_n, tanh=True)
    assert (dgates[..., hidden:].cpu().numpy() != 0)[np.abs(gates[..., hidden:]) < 30].all()


def test_a_device_without_room_for_large_clusters():
    """32 channels and a long axis take clusters of 16 blocks where the device places
    them, and otherwise of 8: the call works, and within the same bounds."""
    import ctypes

    from jstorch_b200 import _lib
    rng = np.random.default_rng(5)
    gates = rng.standard_normal((1500, 1, 64)).astype(np.float32)
    h0, dh_n = (rng.standard_normal((1, 32)).astype(np.float32) for _ in range(2))
    dout = rng.standard_normal((1500, 1, 32)).astype(np.float32)
    limit = _lib.load().jst_test_scan_cluster
    limit.argtypes, limit.restype = [ctypes.c_int], None
    try:
        for blocks in (16, 8):
            limit(blocks)
            for tanh in (False, True):
                _check(gates, h0, dout, dh_n, tanh=tanh)
    finally:
        limit(16)


# every form with lengths: one lane an axis, two channels a lane in rows of several sequences, small blocks,
# doubled clusters, the backward pass's blocks of four warps, one channel a lane
@pytest.mark.parametrize("seq,batch,hidden", [(9, 5, 64), (16, 300, 6), (70, 40, 64), (90, 333, 10), (33, 300, 130), (64, 700, 60),
                                              (1100, 6, 512), (1000, 40, 256), (1100, 40, 256), (2500, 2, 700), (40, 400, 51), (20, 128, 1024)])
@pytest.mark.parametrize("reverse,tanh", [(False, True), (True, False)])
def test_lengths_in_every_form(seq, batch, hidden, reverse, tanh):
    """Sequences of no step, one, some and all, whose ends fall inside a tile, with anything behind them."""
    rng = np.random.default_rng([seq, batch, hidden])
    lengths = rng.integers(0, seq + 1, batch).astype(np.int32)
    lengths[:5] = [seq, 0, 1, seq - 1, seq // 2][:batch]
    gates = rng.standard_normal((seq, batch, 2 * hidden), dtype=np.float32)
    gates[..., :hidden] += 2 * rng.standard_normal(hidden, dtype=np.float32)
    dout = rng.standard_normal((seq, batch, hidden), dtype=np.float32)
    behind = np.arange(seq)[:, None] >= lengths
    gates[behind] = np.resize(np.array([np.nan, np.inf, -np.inf, 3e38], np.float32), 2 * hidden)
    dout[behind] = np.nan
    h0, dh_n = (rng.standard_normal((batch, hidden), dtype=np.float32) for _ in range(2))
    out, h_n, dgates, dh0 = _check(gates, h0, dout, dh_n, reverse, tanh, lengths)
    none = lengths == 0
    assert np.array_equal(h_n.cpu().numpy()[none], h0[none]) and np.array_equal(dh0.cpu().numpy()[none], dh_n[none])
    assert not out.cpu().numpy()[behind].any() and not dgates.cpu().numpy()[behind].any()
