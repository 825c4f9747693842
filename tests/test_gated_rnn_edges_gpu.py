"""rnn.GatedRNN: degenerate sizes and arguments."""
import pytest

pytestmark = pytest.mark.gpu


def test_no_input_features():
    """Gates are the bias alone; the gradients of the empty weight are empty."""
    import torch
    from jstorch_b200 import rnn
    model = rnn.GatedRNN(0, 5, 2)
    x = torch.zeros((4, 3, 0), device="cuda")
    gates = model.params["bias_l0"].expand(4, 3, 10).contiguous()
    first, _ = rnn.gated_scan(gates)
    one = rnn.GatedRNN(5, 5)
    one.load_state_dict({k.replace("l1", "l0"): v for k, v in model.params.items() if "l1" in k})
    want = one(first)
    out, h_n = model(x)
    assert torch.equal(out, want[0]) and torch.equal(h_n[1], want[1][0])
    out, _, ctx = model.forward_train(x)
    dx, _ = model.backward(ctx, torch.ones_like(out))
    assert dx.shape == x.shape and model.grads["weight_l0"].shape == (10, 0)
    o1, _, c1 = one.forward_train(first)
    dfirst, _ = one.backward(c1, torch.ones_like(o1))
    dgates, _ = rnn.gated_scan_backward(gates, first, dfirst)
    assert (model.grads["bias_l0"] - dgates.sum((0, 1))).abs().max() <= 1e-5
    assert torch.equal(model.quantize()(x)[1][0], h_n[0])


def test_lengths_of_another_kind():
    import torch
    from jstorch_b200 import rnn
    model, x = rnn.GatedRNN(4, 6), torch.zeros((3, 2, 4), device="cuda")
    for call in (model, model.forward_train):
        with pytest.raises(TypeError, match="lengths"):
            call(x, None, [3, 1])
