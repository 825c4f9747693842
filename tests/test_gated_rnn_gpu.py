"""rnn.GatedRNN: projection, scan and dropout run together as a training step,
and 8-bit projections with one scan step at a time as a serving loop, against
the same model written out in torch fp64.

Bounds.  A projection of K terms is off by the fp32 path's 2e-6 of its row
norms; the gates then move a state by at most 1/4 (sigmoid) and 1 (tanh) of
that, averaged over the steps that the state remembers, and every layer passes
its input's error on with the weight's gain.  With the sizes here (weights
uniform within 1/sqrt(K), so a gain below one, three layers at most) outputs
stay within 2e-5 and gradients within 1e-4 of their largest entry: ten times
what the terms above add up to, as for the GRU."""
import numpy as np
import pytest

from oracle import oracle

pytestmark = pytest.mark.gpu


def _reference(model, x, h0, lengths, masks):
    """The model in fp64 torch; masks: the dropout multipliers between layers."""
    import torch
    H, dirs = model.hidden_size, 2 if model.bidirectional else 1
    params = {k: v.double().cpu().requires_grad_() for k, v in model.params.items()}
    inp, h_n = x, []
    for l in range(model.num_layers):
        halves = []
        for d, sfx in enumerate(("", "_reverse")[:dirs]):
            gates = inp @ params[f"weight_l{l}{sfx}"].T + params[f"bias_l{l}{sfx}"]
            h = h0[l * dirs + d]
            outs = [None] * x.shape[0]
            for t in (range(x.shape[0] - 1, -1, -1) if d else range(x.shape[0])):
                z = torch.sigmoid(gates[t, :, :H])
                n = gates[t, :, H:]
                n = torch.tanh(n) if model.candidate == "tanh" else n
                k = (t < lengths)[:, None]
                h = torch.where(k, z * h + (1 - z) * n, h)
                outs[t] = torch.where(k, h, torch.zeros_like(h))
            halves.append(torch.stack(outs))
            h_n.append(h)
        out = torch.cat(halves, dim=2)
        inp = out * masks[l] if l < model.num_layers - 1 else out
    return out, torch.stack(h_n), params


def _near(got, want, tol):
    got, want = got.detach().cpu().double(), want.detach()
    assert got.shape == want.shape
    scale = max(1.0, float(want.abs().max()))
    assert float((got - want).abs().max()) <= tol * scale


@pytest.mark.parametrize("layers,bidir,batch_first,candidate,p", [
    (1, False, False, "tanh", 0.0), (2, True, False, "tanh", 0.3), (3, False, True, "identity", 0.5)])
def test_training_step(layers, bidir, batch_first, candidate, p):
    import torch
    from jstorch_b200.rnn import GatedRNN
    seq, batch, inp, H = 23, 5, 12, 18
    gen = torch.Generator(device="cuda").manual_seed(layers)
    model = GatedRNN(inp, H, layers, bidir, batch_first, candidate, generator=gen, dropout=p, seed=77)
    dirs = 2 if bidir else 1
    rng = np.random.default_rng(layers)
    x = torch.from_numpy(rng.standard_normal((seq, batch, inp)).astype(np.float32))
    h0 = torch.from_numpy(rng.standard_normal((layers * dirs, batch, H)).astype(np.float32))
    dout = torch.from_numpy(rng.standard_normal((seq, batch, H * dirs)).astype(np.float32))
    dh_n = torch.from_numpy(rng.standard_normal((layers * dirs, batch, H)).astype(np.float32))
    lengths = torch.tensor([23, 0, 7, 22, 1], dtype=torch.int32)
    order = (lambda t: t.transpose(0, 1)) if batch_first else (lambda t: t)
    for call in range(2):  # the second pass has other masks, and adds to the gradients
        masks = [torch.from_numpy(oracle.dropout_f32(np.ones((seq, batch, H * dirs), np.float32), p, 77, call * layers + l)).double()
                 if p else 1.0 for l in range(layers)]
        xr, hr = x.double().requires_grad_(), h0.double().requires_grad_()
        want, want_h, params = _reference(model, xr, hr, lengths, masks)
        ((want * dout).sum() + (want_h * dh_n).sum()).backward()
        out, h_n, ctx = model.forward_train(order(x).cuda(), h0.cuda(), lengths.cuda())
        model.zero_grad()
        dx, dh0 = model.backward(ctx, order(dout).cuda(), dh_n.cuda())
        _near(order(out), want, 2e-5)
        _near(h_n, want_h, 2e-5)
        _near(order(dx), xr.grad, 1e-4)
        _near(dh0, hr.grad, 1e-4)
        for k, v in params.items():
            _near(model.grads[k], v.grad, 1e-4)
    before = {k: v.clone() for k, v in model.grads.items()}
    model.backward(ctx, order(dout).cuda(), dh_n.cuda())
    assert all(torch.equal(model.grads[k], before[k] + before[k]) for k in before)


@pytest.mark.parametrize("batch_first", [False, True])
def test_padding_does_not_reach_the_gradients(batch_first):
    """Infinities and NaN behind the sequences, in x and in dout, give the gradients that zeros give."""
    import torch
    from jstorch_b200.rnn import GatedRNN
    model = GatedRNN(9, 11, 2, True, batch_first, dropout=0.25)
    lengths = torch.tensor([6, 0, 3], dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    x, dout = (torch.randn((3, 6, n), generator=gen, device="cuda") for n in (9, 22))
    behind = (torch.arange(6, device="cuda") >= lengths[:, None])[..., None]
    results = []
    for fill in (0.0, float("nan"), float("inf")):
        model.calls, model.grads = 0, {}
        a, b = (torch.where(behind, torch.full_like(t, fill), t) for t in (x, dout))
        if not batch_first:
            a, b = a.transpose(0, 1), b.transpose(0, 1)
        given = a.clone()
        out, h_n, ctx = model.forward_train(a, None, lengths)
        dx, _ = model.backward(ctx, b)
        assert torch.equal(a.nan_to_num(), given.nan_to_num())  # x is the caller's
        results.append([out, h_n, dx, *model.grads.values()])
    for other in results[1:]:
        assert all(torch.equal(r, w) for r, w in zip(other, results[0]))


def test_gradients_against_differences():
    """dL along a direction of every parameter, against (L(+s) - L(-s)) / 2s in
    fp32: each L rounds to 2e-6 of the sum of its terms' magnitudes, over 2s."""
    import torch
    from jstorch_b200.rnn import GatedRNN
    gen = torch.Generator(device="cuda").manual_seed(4)
    model = GatedRNN(9, 14, 2, generator=gen, dropout=0.25, seed=3)
    x, dout = (torch.randn((11, 4, n), device="cuda", generator=gen) for n in (9, 14))
    out, _, ctx = model.forward_train(x)
    model.backward(ctx, dout)
    for k, v in model.params.items():
        way = torch.randn(v.shape, device="cuda", generator=gen)
        losses, step = [], 1e-2
        for s in (step, -step):
            v += s * way
            model.calls = 0
            o = model.forward_train(x)[0].double()
            losses.append(float((o * dout.double()).sum()))
            v -= s * way
        slope = (losses[0] - losses[1]) / (2 * step)
        want = float((model.grads[k].double() * way.double()).sum())
        # curvature: third derivatives of a state are below the direction's cube; rounding: 2e-6 of the terms
        size = float(way.norm()) ** 3 * step ** 2 * float(dout.abs().sum()) / 50
        assert abs(slope - want) <= size + 2e-6 * float((o * dout.double()).abs().sum()) / step, k


def test_serving_loop():
    """Steps of one token each, in fp32 and on 8-bit weights, are the layer run over the whole sequence."""
    import torch
    from jstorch_b200.rnn import GatedRNN
    gen = torch.Generator(device="cuda").manual_seed(8)
    model = GatedRNN(40, 64, 2, generator=gen, dropout=0.5)
    x = torch.randn((12, 3, 40), device="cuda", generator=gen)
    whole, h_whole = model(x)
    h = torch.zeros((2, 3, 64), device="cuda")
    got = torch.stack([model.step(t, h).clone() for t in x])
    _near(got, whole.cpu().double(), 2e-5)
    _near(h, h_whole.cpu().double(), 2e-5)
    model.quantize()
    whole8, h8 = model(x)
    h = torch.zeros((2, 3, 64), device="cuda")
    got = torch.stack([model.step(t, h).clone() for t in x])
    # the first layer's projections are equal row by row; its states differ by a few ulp between the whole scan and
    # single steps, which can move a value of the second layer's input across a rounding border: one step of 1/127 of
    # a token's peak (1) times the channel's largest weight (1/8), for a few of the 64 values: 64 / 127 / 8 at the very most
    assert float((got - whole8).abs().max()) <= 64 / 127 / 8
    assert float((got - whole8).abs().mean()) <= 1e-4
    # against fp32: a weight and an input are each off by half a step of their peak / 127, K terms of random sign
    assert float((whole8 - whole).abs().mean()) <= 2 * (0.5 / 127) * 3
    # the 8-bit model written out: oracle products, the oracle's scan
    q, s = (t.cpu().numpy() for t in model.quantized["weight_l0"])
    xq, xs = oracle.quantize_rows(x.cpu().numpy().reshape(36, 40))
    gates = oracle.gemm_i8_f64(xq, q, xs, s, model.params["bias_l0"].cpu().numpy())[0].reshape(12, 3, 128)
    one = GatedRNN(40, 64)
    one.load_state_dict({k: v for k, v in model.params.items() if "l0" in k})
    got, _ = one.quantize()(x)
    _near(got, torch.from_numpy(oracle.scan_f64(gates)["out"][0]), 2e-5)


def test_captured_training_step_beside_an_eager_one():
    import torch
    from jstorch_b200.rnn import GatedRNN
    gen = torch.Generator(device="cuda").manual_seed(2)
    model = GatedRNN(16, 24, 2, generator=gen, dropout=0.2)
    x, dout = torch.randn((9, 4, 16), device="cuda", generator=gen), torch.randn((9, 4, 24), device="cuda", generator=gen)
    out, _, ctx = model.forward_train(x)
    dx, _ = model.backward(ctx, dout)
    want = {k: v.clone() for k, v in model.grads.items()}
    graph = torch.cuda.CUDAGraph()
    model.zero_grad()
    torch.cuda.synchronize()
    model.calls = 0
    with torch.cuda.graph(graph):
        out_g, _, ctx_g = model.forward_train(x)
        dx_g, _ = model.backward(ctx_g, dout)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out_g, out) and torch.equal(dx_g, dx)
    assert all(torch.equal(model.grads[k], want[k]) for k in want)


@pytest.mark.parametrize("seq,batch", [(0, 3), (4, 0), (1, 1)])
def test_small(seq, batch):
    import torch
    from jstorch_b200.rnn import GatedRNN
    model = GatedRNN(5, 7, 2, dropout=0.1)
    x = torch.randn((seq, batch, 5), device="cuda")
    out, h_n, ctx = model.forward_train(x)
    dx, dh0 = model.backward(ctx, torch.ones_like(out))
    assert out.shape == (seq, batch, 7) and h_n.shape == (2, batch, 7) and dx.shape == x.shape and dh0 is None
    assert model.quantize()(x)[0].shape == out.shape


def test_refusals():
    import torch
    from jstorch_b200.rnn import GRU, GatedRNN
    with pytest.raises(ValueError):
        GatedRNN(4, 4, candidate="relu")
    with pytest.raises(ValueError):
        GatedRNN(4, 4, dropout=1.5)
    with pytest.raises(ValueError):
        GRU(4, 4, dropout=-0.5)
    model = GatedRNN(4, 6, bidirectional=True)
    x = torch.zeros((3, 2, 4), device="cuda")
    for call in (lambda: model(x[0]), lambda: model(x[..., :3]), lambda: model(x, torch.zeros((1, 2, 6), device="cuda")),
                 lambda: model.step(x[0], torch.zeros((2, 2, 6), device="cuda")),
                 lambda: model.forward_train(x, None, torch.zeros(3, dtype=torch.int32, device="cuda")),
                 lambda: model.forward_train(x, None, torch.zeros(2, dtype=torch.int32)),
                 lambda: model.load_state_dict({"bias_l0": torch.zeros(3)}),
                 lambda: GatedRNN(4, 6).step(x[0], torch.zeros((1, 3, 6), device="cuda"))):
        with pytest.raises(ValueError):
            call()
