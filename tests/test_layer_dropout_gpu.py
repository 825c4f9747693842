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
