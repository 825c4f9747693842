"""The cases that measure three families of operators, and their plain forms.

  linear_i8 / gemm_i8   an 8-bit integer matrix product with one scale a token and one a channel.
                        kind "linear": fp32 rows are quantised on the way (q = round(x / s), s = max|x| / 127 a row);
                        kind "gemm": the rows are quantised already.
                            y[m, n] = relu?(s[m] * sw[n] * sum_k q[m, k] * w[n, k] + bias[n])
  gated_scan            a gated linear recurrence over time, channel by channel, from pre-activations (a | c):
                            z = sigmoid(a)    n = tanh(c) or c    h_t = z_t * h_{t-1} + (1 - z_t) * n_t
                        kind "scan": the forward pass; kind "scan_train": the forward pass and the gradients.
  dropout               y = x * [r >= p * 2^32] / (1 - p), r the words of Philox4x32-10 at the element's index;
                        kind "dropout": one pass; kind "dropout_train": the pass and its gradient (the same mask again).

`own` chooses who computes: False, the plain forms below; True, the package's operators.
"""
import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token through one 8-bit layer of the 8192 x 8192 benchmark's width: a serving step, bound by the weight
        {"name": "linear 1x8192x8192", "kind": "linear", "m": 1, "n": 8192, "k": 8192, "bias": False, "relu": False},
        # a handful of sequences decoding together through the recurrent benchmark's input projection (512 -> 2 x 1024)
        {"name": "linear 5x2048x512", "kind": "linear", "m": 5, "n": 2048, "k": 512, "bias": True, "relu": False},
        # the first layer of the 784-1024-1024-10 network at batch 256, with its bias and ReLU
        {"name": "linear 256x1024x784", "kind": "linear", "m": 256, "n": 1024, "k": 784, "bias": True, "relu": True},
        # a long prompt through a wide layer: the largest product
        {"name": "gemm 8192x8192x8192", "kind": "gemm", "m": 8192, "n": 8192, "k": 8192, "bias": False, "relu": False},
        # sizes that fit no tile, rows padded to 16 bytes as the quantiser leaves them
        {"name": "gemm 1001x1537x2043", "kind": "gemm", "m": 1001, "n": 1537, "k": 2043, "bias": True, "relu": False},
        # one time step of one sequence: the smallest call of a serving loop
        {"name": "scan 1x1x1024", "kind": "scan", "seq": 1, "batch": 1, "hidden": 1024, "h0": True, "ragged": False,
         "reverse": False, "tanh": True},
        # the recurrent benchmark's layer: 64 steps of 64 sequences, 1024 units
        {"name": "scan 64x64x1024", "kind": "scan", "seq": 64, "batch": 64, "hidden": 1024, "h0": False, "ragged": False,
         "reverse": False, "tanh": True},
        # one long document: few channels, so the time axis has to be split
        {"name": "scan 65536x1x1024", "kind": "scan", "seq": 65536, "batch": 1, "hidden": 1024, "h0": True,
         "ragged": False, "reverse": False, "tanh": False},
        # a training step over a padded batch of documents
        {"name": "train 2048x16x1024", "kind": "scan_train", "seq": 2048, "batch": 16, "hidden": 1024, "h0": True,
         "ragged": True, "reverse": False, "tanh": True},
        # the backward direction of a bidirectional layer at odd sizes
        {"name": "train 777x3x333", "kind": "scan_train", "seq": 777, "batch": 3, "hidden": 333, "h0": True,
         "ragged": True, "reverse": True, "tanh": True},
        # between two recurrent layers: 64 steps of 64 sequences, 1024 units
        {"name": "dropout 4096x1024", "kind": "dropout", "rows": 4096, "cols": 1024, "p": 0.1},
        # forward and backward over an activation of the 8192 x 8192 benchmark's size
        {"name": "dropout 8192x8192", "kind": "dropout_train", "rows": 8192, "cols": 8192, "p": 0.25},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "gemm", "scan", "scan_train", "dropout", "dropout_train"])
    if kind in ("linear", "gemm"):
        return {"kind": kind, "m": _log(rng, 1, 8192), "n": _log(rng, 1, 8192), "k": _log(rng, 1, 8192),
                "bias": rng.random() < 0.5, "relu": rng.random() < 0.5}
    if kind.startswith("scan"):
        most = 1 << 25 if kind == "scan_train" else 1 << 26  # elements: what the largest listed case of the kind has
        hidden = _log(rng, 1, 4096)
        seq = _log(rng, 1, min(65536, most // hidden))
        batch = _log(rng, 1, max(1, min(512, most // (hidden * seq))))
        return {"kind": kind, "seq": seq, "batch": batch, "hidden": hidden, "h0": rng.random() < 0.5,
                "ragged": rng.random() < 0.5, "reverse": rng.random() < 0.5, "tanh": rng.random() < 0.5}
    return {"kind": kind, "rows": _log(rng, 1, 8192), "cols": _log(rng, 1, 8192), "p": round(rng.uniform(0.0, 0.9), 3)}


# ------------------------------------------------------------------ the inputs
def _pitched(values):
    """Rows 16 bytes aligned, as the quantiser lays 8-bit rows out."""
    rows, cols = values.shape
    held = torch.zeros((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=values.device)
    held[:, :cols] = values
    return held[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    s = {"case": case}
    if case["kind"] in ("linear", "gemm"):
        m, n, k = case["m"], case["n"], case["k"]
        # weights of variance 1 / k whose channels differ in size, quantised channel by channel
        w = randn(n, k) * torch.exp(0.5 * randn(n, 1)) / math.sqrt(k)
        s["w_scale"] = (w.abs().amax(1).double() / 127).float()
        s["w"] = _pitched(torch.round(w.double() / s["w_scale"].double()[:, None]).clamp(-127, 127).to(torch.int8))
        s["bias"] = 0.1 * randn(n) if case["bias"] else None
        x = randn(m, k) * torch.exp(0.5 * randn(m, 1))  # tokens of different size
        if case["kind"] == "linear":
            s["x"] = x
        else:
            s["x_scale"] = (x.abs().amax(1).double() / 127).float()
            s["x"] = _pitched(torch.round(x.double() / s["x_scale"].double()[:, None]).clamp(-127, 127).to(torch.int8))
        return s
    if case["kind"].startswith("scan"):
        seq, batch, hidden = case["seq"], case["batch"], case["hidden"]
        gates = randn(seq, batch, 2 * hidden)
        gates[..., :hidden] += 2.0 * randn(hidden)  # channels that forget at once and channels that remember for long
        s["gates"] = gates
        s["h0"] = randn(batch, hidden) if case["h0"] else None
        s["lengths"] = None
        if case["ragged"]:
            s["lengths"] = torch.randint(0, seq + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
            s["lengths"][0] = seq
        if case["kind"] == "scan_train":
            s["dout"], s["dh_n"] = randn(seq, batch, hidden), randn(batch, hidden)
        return s
    s["x"] = randn(case["rows"], case["cols"])
    s["seed"], s["offset"] = (seed * 0x9E3779B97F4A7C15 + 1) % (1 << 63), seed % 1000
    if case["kind"] == "dropout_train":
        s["dy"] = randn(case["rows"], case["cols"])
    return s


# ------------------------------------------------------------------ plain forms
def _plain_product(s):
    case, x = s["case"], s["x"]
    if case["kind"] == "linear":
        scale = x.abs().amax(1) / 127
        # in 64 bits: a quotient next to a half goes to the side that it lies on
        q = torch.where(scale[:, None] > 0, torch.round(x.double() / scale.double()[:, None]), 0.0).clamp(-127, 127)
    else:
        scale, q = s["x_scale"], x.double()
    # sums of up to 8192 products of 127 * 127 pass 2^24: 64 bits hold them
    y = torch.matmul(q, s["w"].double().t()) * (scale.double()[:, None] * s["w_scale"].double())
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if case["relu"]:
        y = torch.where(y > 0, y, torch.zeros_like(y))
    return y.float()


def _plain_scan_of(a, b):
    """h_t = a_t * h_{t-1} + b_t along the first axis from h_{-1} = 0: pairs (a, b) composed over doubling distances."""
    d = 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _plain_gates(s):
    """(z, n, valid) in time order of the recurrence (flipped for a reverse one); a step outside its sequence keeps the state."""
    case, hidden = s["case"], s["case"]["hidden"]
    gates = s["gates"].flip(0) if case["reverse"] else s["gates"]
    a, c = gates[..., :hidden], gates[..., hidden:]
    t = torch.arange(case["seq"], device=a.device)
    if case["reverse"]:
        t = t.flip(0)
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((case["batch"],), case["seq"], device=a.device)
    valid = (t[:, None] < lengths[None, :])[..., None]
    e = torch.exp(-a.abs())
    big, small = 1 / (1 + e), e / (1 + e)  # sigmoid(|a|) and sigmoid(-|a|), each to its last bits
    z = torch.where(a >= 0, big, small)
    rest = torch.where(a >= 0, small, big)  # 1 - z
    n = torch.tanh(c) if case["tanh"] else c
    return z, rest, n, valid


def _plain_scan(s):
    case = s["case"]
    z, rest, n, valid = _plain_gates(s)
    one, zero = torch.ones_like(z), torch.zeros_like(z)
    keep, add = torch.where(valid, z, one), torch.where(valid, rest * n, zero)
    h0 = s["h0"] if s["h0"] is not None else torch.zeros_like(add[0])
    state = _plain_scan_of(torch.cat([one[:1], keep]), torch.cat([h0[None], add]))  # h_{-1}, h_0, ...
    out = torch.where(valid, state[1:], zero)
    h_n = state[-1].clone()
    if case["kind"] == "scan":
        return {"out": out.flip(0) if case["reverse"] else out, "h_n": h_n}
    # G_t = dL/dh_t: what the output gives and what the next step hands back
    dout = s["dout"].flip(0) if case["reverse"] else s["dout"]
    give = torch.where(valid, dout, zero)
    # G_t = keep_{t+1} * G_{t+1} + give_t, the last one with dh_n
    back_a = torch.cat([one[:1], keep.flip(0)[:-1]])
    back_b = give.flip(0).clone()
    back_b[0] += s["dh_n"]
    total = _plain_scan_of(back_a, back_b).flip(0)
    before = state[:-1]
    dz, dn = total * (before - n), total * rest
    da = torch.where(valid, dz * z * rest, zero)
    dc = torch.where(valid, dn * (1 - n * n) if case["tanh"] else dn, zero)
    dgates = torch.cat([da, dc], dim=2)
    if case["reverse"]:
        out, dgates = out.flip(0), dgates.flip(0)
    r = {"out": out, "h_n": h_n, "dgates": dgates}
    if s["h0"] is not None:
        r["dh0"] = keep[0] * total[0]
    return r


def _plain_words(count, seed, offset, device):
    """Words of Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): counter (index // 4, offset), key = seed."""
    low = 0xFFFFFFFF
    c0 = torch.arange((count + 3) // 4, dtype=torch.int64, device=device)
    c1, c2, c3 = c0 >> 32, torch.full_like(c0, offset & low), torch.full_like(c0, offset >> 32)
    c0 = c0 & low
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # products modulo 2^64: both halves are right
        c0, c1, c2, c3 = ((q >> 32) & low) ^ c1 ^ k0, q & low, ((p >> 32) & low) ^ c3 ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:count]


def _plain_dropout(s):
    case, x = s["case"], s["x"]
    p = case["p"]
    keep = (_plain_words(x.numel(), s["seed"], s["offset"], x.device) >= int(p * 4294967296.0)).reshape(x.shape)
    scale = torch.tensor(1.0 / (1.0 - p), dtype=torch.float32, device=x.device)
    zero = torch.zeros((), dtype=torch.float32, device=x.device)
    y = torch.where(keep, x * scale, zero)
    if case["kind"] == "dropout":
        return {"y": y}
    return {"y": y, "dx": torch.where(keep, s["dy"] * scale, zero)}


# ------------------------------------------------------------------ one pass
def _own(s):
    import jstorch_b200
    from jstorch_b200 import quant, rnn

    case = s["case"]
    if case["kind"] == "linear":
        return quant.linear_i8(s["x"], s["w"], s["w_scale"], bias=s["bias"], relu=case["relu"])
    if case["kind"] == "gemm":
        return quant.gemm_i8(s["x"], s["w"], s["x_scale"], s["w_scale"], bias=s["bias"], relu=case["relu"])
    if case["kind"].startswith("scan"):
        how = {"lengths": s["lengths"], "reverse": case["reverse"], "candidate": "tanh" if case["tanh"] else "identity"}
        out, h_n = rnn.gated_scan(s["gates"], s["h0"], **how)
        if case["kind"] == "scan":
            return {"out": out, "h_n": h_n}
        dgates, dh0 = rnn.gated_scan_backward(s["gates"], out, s["dout"], s["h0"], dh_n=s["dh_n"], **how)
        r = {"out": out, "h_n": h_n, "dgates": dgates}
        if dh0 is not None:
            r["dh0"] = dh0
        return r
    y = jstorch_b200.dropout(s["x"], case["p"], s["seed"], s["offset"])
    if case["kind"] == "dropout":
        return {"y": y}
    return {"y": y, "dx": jstorch_b200.dropout(s["dy"], case["p"], s["seed"], s["offset"])}


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind in ("linear", "gemm"):
        return _plain_product(state)
    return _plain_scan(state) if kind.startswith("scan") else _plain_dropout(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] in ("linear", "gemm"):
        m, n, k = case["m"], case["n"], case["k"]
        x = 4 * m * k if case["kind"] == "linear" else m * k + 4 * m
        return {"bytes": x + n * k + 4 * n + (4 * n if case["bias"] else 0) + 4 * m * n, "flops": 2 * m * n * k}
    if case["kind"].startswith("scan"):
        steps = case["seq"] * case["batch"] * case["hidden"]
        edge = 4 * case["batch"] * case["hidden"]
        # of a padded batch the steps inside the sequences are read, half of them on average; every output place is written
        read = steps / 2 * (1 + 1 / case["batch"]) if case["ragged"] else steps
        if case["kind"] == "scan":
            return {"bytes": 8 * read + 4 * steps + edge * (2 if case["h0"] else 1), "flops": 10 * read}
        return {"bytes": 12 * read + 12 * steps + edge * (4 if case["h0"] else 2), "flops": 30 * read}
    n = case["rows"] * case["cols"]
    return {"bytes": 8 * n, "flops": n} if case["kind"] == "dropout" else {"bytes": 16 * n, "flops": 2 * n}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_product(s):
    case = s["case"]
    x = s["x"].to(torch.float64)
    if case["kind"] == "linear":
        peak = torch.max(torch.max(x, -x), dim=1).values
        scale = (peak / 127).to(torch.float32).to(torch.float64)  # the scale is a 32-bit number by definition
        x = torch.round(x / torch.where(scale == 0, torch.ones_like(scale), scale).unsqueeze(1))
    else:
        scale = s["x_scale"].to(torch.float64)
    y = torch.einsum("mk,nk->mn", x, s["w"].to(torch.float64))
    y = y * scale.unsqueeze(1) * s["w_scale"].to(torch.float64).unsqueeze(0)
    if s["bias"] is not None:
        y = y + s["bias"].to(torch.float64).unsqueeze(0)
    return torch.clamp(y, min=0.0) if case["relu"] else y


def _exact_scan(s):
    case, hidden = s["case"], s["case"]["hidden"]
    gates = s["gates"].to(torch.float64)
    z = 1 / (1 + torch.exp(-gates[..., :hidden]))
    n = torch.tanh(gates[..., hidden:]) if case["tanh"] else gates[..., hidden:]
    lengths = [case["seq"]] * case["batch"] if s["lengths"] is None else s["lengths"].tolist()
    times = list(range(case["seq"]))
    if case["reverse"]:
        times.reverse()
    inside = torch.tensor([[[t < length] for length in lengths] for t in range(case["seq"])], device=z.device) if case["ragged"] else None
    h = torch.zeros_like(z[0]) if s["h0"] is None else s["h0"].to(torch.float64)
    before, out = torch.empty_like(z), torch.zeros_like(z)
    for t in times:  # step by step, as the recurrence is written
        before[t] = h
        new = n[t] + z[t] * (h - n[t])
        h = new if inside is None else torch.where(inside[t], new, h)
        out[t] = h if inside is None else h * inside[t]
    r = {"out": out, "h_n": h}
    if case["kind"] == "scan":
        return r
    g, dgates = s["dh_n"].to(torch.float64), torch.zeros_like(gates)
    for t in reversed(times):
        mine = g + s["dout"][t].to(torch.float64)
        da = mine * (before[t] - n[t]) * z[t] * (1 - z[t])
        dc = mine * (1 - z[t]) * (1 - n[t] ** 2 if case["tanh"] else 1.0)
        both = torch.cat([da, dc], dim=1)
        dgates[t] = both if inside is None else both * inside[t]
        g = z[t] * mine if inside is None else torch.where(inside[t], z[t] * mine, g)
    r["dgates"] = dgates
    if s["h0"] is not None:
        r["dh0"] = g
    return r


def _exact_dropout(s):
    case, x = s["case"], s["x"]
    total, p = x.numel(), case["p"]
    kept = np.empty(total, dtype=bool)
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    threshold, chunk = np.uint64(math.floor(p * 2.0 ** 32)), 1 << 20
    for first in range(0, (total + 3) // 4, chunk):
        block = np.arange(first, min(first + chunk, (total + 3) // 4), dtype=np.uint64)
        word = [block & low, block >> shift, np.full_like(block, s["offset"] % 2 ** 32), np.full_like(block, s["offset"] // 2 ** 32)]
        key = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32]
        for _ in range(10):
            left, right = np.uint64(0xD2511F53) * word[0], np.uint64(0xCD9E8D57) * word[2]
            word = [(right >> shift) ^ word[1] ^ np.uint64(key[0]), right & low, (left >> shift) ^ word[3] ^ np.uint64(key[1]), left & low]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        words = np.stack(word, axis=1).reshape(-1)
        kept[4 * first: 4 * first + len(words)] = (words >= threshold)[: total - 4 * first]
    keep = torch.from_numpy(kept).to(x.device).reshape(x.shape)

    def of(v):
        return torch.where(keep, v.to(torch.float64) / (1.0 - p), torch.zeros((), dtype=torch.float64, device=v.device))

    return {"y": of(x)} if case["kind"] == "dropout" else {"y": of(x), "dx": of(s["dy"])}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("linear", "gemm"):
        return _exact_product(s)
    return _exact_scan(s) if case["kind"].startswith("scan") else _exact_dropout(s)
