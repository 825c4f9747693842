"""The masks of rnn.GRU's and rnn.GatedRNN's dropout, pass by pass."""
import pytest

pytestmark = pytest.mark.gpu


def _model(kind, seed=5):
    import torch
    from jstorch_b200 import rnn
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return getattr(rnn, kind)(6, 10, 3, generator=gen, dropout=0.4, seed=11), torch.randn((7, 3, 6), device="cuda", generator=gen)


@pytest.mark.parametrize("kind", ["GRU", "GatedRNN"])
def test_a_refused_pass_takes_no_masks(kind):
    """A training pass after a refused one draws what it would have drawn without it."""
    import torch
    model, x = _model(kind)
    other, _ = _model(kind)
    h0 = torch.zeros((3, 3, 10), device="cuda")
    refused = [lambda: model.forward_train(x, h0[:, :2]), lambda: model.forward_train(x.double())]
    if kind == "GatedRNN":
        refused += [lambda: model.forward_train(x, h0.double()),
                    lambda: model.forward_train(x, None, torch.zeros(3, dtype=torch.int64, device="cuda"))]
    for call in refused:
        with pytest.raises((ValueError, TypeError)):
            call()
    for _ in range(2):
        assert torch.equal(model.forward_train(x)[0], other.forward_train(x)[0])


@pytest.mark.parametrize("kind", ["GRU", "GatedRNN"])
def test_masks_of_a_captured_step(kind):
    """Replays of one captured pass, forward and gradients, are eager passes one after the other."""
    import torch
    model, x = _model(kind)
    other, _ = _model(kind)
    dout = torch.randn_like(model(x)[0])
    out, _, ctx = other.forward_train(x)
    other.backward(ctx, dout)  # makes the gradients' buffers
    model.backward(model.forward_train(x)[2], dout)
    other.calls = model.calls = 0
    model.mask_step = torch.zeros(1, dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        model.zero_grad()
        out, _, ctx = model.forward_train(x)
        dx, _ = model.backward(ctx, dout)
        model.mask_step += model.num_layers
    seen = []
    for _ in range(3):
        graph.replay()
        other.zero_grad()
        want, _, c = other.forward_train(x)
        want_dx, _ = other.backward(c, dout)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(dx, want_dx)
        assert all(torch.equal(model.grads[k], other.grads[k]) for k in other.grads)
        seen.append(out.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
