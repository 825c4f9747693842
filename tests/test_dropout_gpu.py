"""jstorch_b200.dropout against the generator written out in numpy: the mask
and the values are equal bit for bit (x times one fp32 number is rounded once
on either side)."""
import numpy as np
import pytest

from oracle import oracle

pytestmark = pytest.mark.gpu
SEED, OFFSET = 0x9E3779B97F4A7C15, (7 << 32) + 5


def _equal(got, x, p, seed=SEED, offset=OFFSET):
    np.testing.assert_array_equal(got.cpu().numpy(), oracle.dropout_f32(x, p, seed, offset))


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 127, 1023, 1024, 1025, 4096, 100003])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_sizes_and_alignments(n, shift):
    import torch

    import jstorch_b200
    x = np.random.default_rng(n).standard_normal(n).astype(np.float32)
    held = torch.zeros(n + 8, device="cuda")
    held[shift:shift + n] = torch.from_numpy(x).cuda()
    _equal(jstorch_b200.dropout(held[shift:shift + n], 0.3, SEED, OFFSET), x, 0.3)
    out = torch.full((n + 8,), 7.0, device="cuda")  # written from another alignment than it is read at
    jstorch_b200.dropout(held[shift:shift + n], 0.3, SEED, OFFSET, out=out[1:1 + n])
    _equal(out[1:1 + n], x, 0.3)
    assert bool((out[:1] == 7).all()) and bool((out[1 + n:] == 7).all())


@pytest.mark.parametrize("n,shift", [(1212416, 0), (1300001, 0), (2500003, 1)])
def test_many_elements(n, shift):
    import torch

    import jstorch_b200
    x = np.random.default_rng(n).standard_normal(n + shift).astype(np.float32)
    _equal(jstorch_b200.dropout(torch.from_numpy(x).cuda()[shift:], 0.6, SEED, OFFSET), x[shift:], 0.6)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -33, 0.1, 0.5, 0.9, 1 - 2.0 ** -24, 1.0])
def test_probabilities(p):
    import torch

    import jstorch_b200
    x = np.random.default_rng(3).standard_normal((50, 40)).astype(np.float32)
    _equal(jstorch_b200.dropout(torch.from_numpy(x).cuda(), p, 1, 0), x, p, 1, 0)


def test_dropped_elements_are_zero_whatever_they_hold():
    import torch

    import jstorch_b200
    x = np.resize(np.array([np.inf, -np.inf, np.nan, 1e-45, 3e38, -0.0], np.float32), 6000)
    y = jstorch_b200.dropout(torch.from_numpy(x).cuda(), 0.5, SEED, OFFSET)
    _equal(y, x, 0.5)
    assert not jstorch_b200.dropout(torch.from_numpy(x).cuda(), 1.0, 1).any()


@pytest.mark.parametrize("rows,cols,ldx,ldy", [(5, 7, 9, 7), (5, 7, 7, 11), (3, 1, 4, 2), (64, 128, 200, 132), (9, 4, 8, 4)])
def test_pitches(rows, cols, ldx, ldy):
    import torch

    import jstorch_b200
    x = np.random.default_rng(rows).standard_normal((rows, cols)).astype(np.float32)
    a, b = torch.zeros((rows, ldx), device="cuda"), torch.full((rows, ldy), 7.0, device="cuda")
    a[:, :cols] = torch.from_numpy(x).cuda()
    jstorch_b200.dropout(a[:, :cols], 0.4, SEED, OFFSET, out=b[:, :cols])
    _equal(b[:, :cols], x, 0.4)
    assert bool((b[:, cols:] == 7).all())
    three = a[:, None, :cols]  # a dimension of one in the middle
    _equal(jstorch_b200.dropout(three, 0.4, SEED, OFFSET)[:, 0], x, 0.4)


def test_in_place_and_backward():
    import torch

    import jstorch_b200
    x, dy = (np.random.default_rng(i).standard_normal(5000).astype(np.float32) for i in (1, 2))
    t = torch.from_numpy(x).cuda()
    assert jstorch_b200.dropout(t, 0.2, 3, 4, out=t) is t
    _equal(t, x, 0.2, 3, 4)
    # the gradient of sum(dy * y) is dy through the same mask: y is linear in x, so a difference is exact up to rounding
    g = jstorch_b200.dropout(torch.from_numpy(dy).cuda(), 0.2, 3, 4)
    _equal(g, dy, 0.2, 3, 4)
    assert torch.equal(g != 0, t != 0)


def test_step_counter_in_a_captured_graph():
    import torch

    import jstorch_b200
    x = np.random.default_rng(1).standard_normal((33, 65)).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = jstorch_b200.dropout(t, 0.5, SEED, OFFSET, step=step)
        step += 1
    for k in range(3):
        g.replay()
        torch.cuda.synchronize()
        _equal(y, x, 0.5, SEED, OFFSET + k)
    step.fill_(-1)  # modulo 2^64
    _equal(jstorch_b200.dropout(t, 0.5, SEED, 0, step=step), x, 0.5, SEED, (1 << 64) - 1)


def test_large_and_other_stream():
    """2^31 + 3 elements: indices past 32 bits draw the words that they should."""
    import torch

    import jstorch_b200
    n = (1 << 31) + 3
    x = torch.ones(n, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = jstorch_b200.dropout(x, 0.5, SEED, OFFSET, out=x, stream=side)
    side.synchronize()
    first = (n // 4 - 1000)
    block = np.arange(first, (n + 3) // 4, dtype=np.uint64)
    one = np.ones_like(block)
    words = oracle.philox4x32_10(np.stack([block, 0 * one, 5 * one, 7 * one], axis=1), (SEED & 0xFFFFFFFF, SEED >> 32))
    keep = (words.reshape(-1) >= 1 << 31)[: n - 4 * first]
    np.testing.assert_array_equal(y[4 * first:].cpu().numpy(), np.where(keep, 2.0, 0.0).astype(np.float32))


def test_empty():
    import torch

    import jstorch_b200
    assert jstorch_b200.dropout(torch.zeros((0, 5), device="cuda"), 0.5, 1).shape == (0, 5)


def test_refusals():
    import torch

    import jstorch_b200
    x = torch.zeros((4, 6), device="cuda")
    bad = [
        lambda: jstorch_b200.dropout(x, 1.5, 1), lambda: jstorch_b200.dropout(x, float("nan"), 1),
        lambda: jstorch_b200.dropout(x, 0.5, -1), lambda: jstorch_b200.dropout(x, 0.5, 1 << 64),
        lambda: jstorch_b200.dropout(x, 0.5, 1, -1), lambda: jstorch_b200.dropout(x.t(), 0.5, 1),
        lambda: jstorch_b200.dropout(x[:, ::2], 0.5, 1), lambda: jstorch_b200.dropout(x[:1].expand(4, 6), 0.5, 1),
        lambda: jstorch_b200.dropout(x, 0.5, 1, out=x[:3]),
        lambda: jstorch_b200.dropout(x, 0.5, 1, step=torch.zeros(1, device="cuda")),
        lambda: jstorch_b200.dropout(x, 0.5, 1, step=torch.zeros(1, dtype=torch.int64)),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    flat = torch.zeros(100, device="cuda")
    with pytest.raises(jstorch_b200.JstError, match="overlap"):
        jstorch_b200.dropout(flat[:50], 0.5, 1, out=flat[1:51])


def test_core_dropout_and_module():
    """Tensor.dropout, its gradient and nn.Dropout of the host core."""
    from jstorch_b200 import _core, nn
    x = np.random.default_rng(4).standard_normal((9, 14)).astype(np.float32)
    t = _core.Tensor.fromBuffer(x)
    np.testing.assert_array_equal(t.dropout(0.3, 5, 6).toArray(), oracle.dropout_f32(x, 0.3, 5, 6))
    np.testing.assert_array_equal(t.transpose().dropout(0.3, 5, 6).toArray(), oracle.dropout_f32(x.T, 0.3, 5, 6))
    g = _core.GradTensor(t, True)
    up = np.random.default_rng(5).standard_normal((9, 14)).astype(np.float32)
    g.dropout(0.3, 5, 6).backward(_core.Tensor.fromBuffer(up))
    np.testing.assert_array_equal(g.grad.toArray(), oracle.dropout_f32(up, 0.3, 5, 6))
    with pytest.raises(RuntimeError, match="dropout"):
        t.dropout(2.0, 1, 1)
    d = nn.Sequential(nn.Dropout(0.3, seed=5))
    for call in range(2):  # a mask of its own for each call
        np.testing.assert_array_equal(d(t).toArray(), oracle.dropout_f32(x, 0.3, 5, call))
    d.eval()
    np.testing.assert_array_equal(d(t).toArray(), x)
    with pytest.raises(ValueError):
        nn.Dropout(-0.1)


def test_gru_dropout_between_layers():
    """A stacked GRU with dropout is its layers run one by one with the dropped
    outputs handed on; its gradients agree with a difference of the loss."""
    import torch

    import jstorch_b200
    from jstorch_b200.rnn import GRU
    gen = torch.Generator(device="cuda").manual_seed(1)
    gru = GRU(6, 10, 2, bidirectional=True, generator=gen, dropout=0.4, seed=11)
    x, dout = (torch.randn((7, 3, n), device="cuda", generator=gen) for n in (6, 20))
    out, h_n, ctx = gru.forward_train(x)
    one, two = GRU(6, 10, 1, bidirectional=True), GRU(20, 10, 1, bidirectional=True)
    one.load_state_dict(gru.params)
    two.load_state_dict({k.replace("l1", "l0"): v for k, v in gru.params.items() if "l1" in k})
    mid = jstorch_b200.dropout(one(x)[0], 0.4, 11, 0)
    assert torch.equal(out, two(mid)[0])
    dx, _ = gru.backward(ctx, dout)
    o1, _, c1 = one.forward_train(x)
    o2, _, c2 = two.forward_train(mid)
    dmid, _ = two.backward(c2, dout)
    want, _ = one.backward(c1, jstorch_b200.dropout(dmid, 0.4, 11, 0))
    assert torch.equal(dx, want)
    assert all(torch.equal(gru.grads[k], one.grads[k]) for k in one.grads)
    again, _, _ = gru.forward_train(x)  # the next call has masks of its own
    assert not torch.equal(again, out)
    assert torch.equal(gru(x)[0], two(one(x)[0])[0])  # serving drops nothing
