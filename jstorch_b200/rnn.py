"""Recurrent layers on torch CUDA tensors: the GRU through jst_gru_layer_forward
(include/jstorch_rnn.h) and a gated linear recurrence (include/jstorch_scan.h).

Mirrors the reference's nn.GRU (src/nn.js:451-536): PyTorch parameter names
(weight_ih_l{l}[_reverse] [3H, in], weight_hh_l{l} [3H, H], bias_ih_l{l},
bias_hh_l{l} [3H]), gate order (r, z, n), num_layers, bidirectional and
batch_first, forward(x, h0=None) -> (output, h_n).

Training: the reference trains the GRU through GradTensor when its
parameters require grad (nn.js:442-444, 477-485; backward through
autograd.hpp:433-441 for the cell's matmuls and the gate ops' closures).
Here forward_train() runs jst_gru_layer_forward_train and keeps the gate
values, and backward(ctx, dout, dh_n) runs jst_gru_layer_backward per layer
and direction, last layer first: parameter gradients accumulate into
self.grads (as .grad does; zero_grad() clears them) and the gradients of x
and h0 are returned.  dropout > 0 drops the output of every layer but the last
in forward_train (include/jstorch_dropout.h); forward() never drops.  Every
pass has masks of its own; in a captured graph, which repeats one pass, they
come from mask_step (a device counter; see _LayerDropout).

gated_scan / gated_scan_backward run the recurrence h_t = z_t h_{t-1} +
(1 - z_t) n_t on given gate pre-activations; GatedRNN is the layer around it
(projection, scan, dropout), with step() and quantize() for serving.
"""
from __future__ import annotations

import ctypes

from . import _lib
from .dropout import dropout as drop
from .gemm import gemm

ACC_DX, ACC_PARAMS, ACC_DH0 = 1, 2, 4  # JST_GRU_ACC_* (include/jstorch_rnn.h)


class _TrainContext:
    """What backward() needs from one forward_train() call."""

    def __init__(self, seq, batch, inps, outs, saved, h0, call=0):
        self.seq, self.batch = seq, batch
        self.inps, self.outs, self.saved, self.h0 = inps, outs, saved, h0
        self.call = call  # number of the forward_train() call: its dropout masks


class _LayerDropout:
    """Dropout between stacked layers: layer l of the model's n-th training
    pass has the mask of (seed, offset n * num_layers + l + *mask_step).

    A captured graph repeats the pass that it was captured in: its masks too,
    unless mask_step, an int64 CUDA tensor of one element on the model's device
    (None: 0), is set before the capture and advanced by num_layers behind the
    pass's backward(), in the graph.  Every replay then draws the masks that the
    next pass would."""

    def _init_dropout(self, dropout: float, seed: int) -> None:
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"dropout must be in [0, 1] (got {dropout})")
        self.dropout, self.seed, self.calls, self.mask_step = dropout, seed, 0, None

    def _drop(self, x, call: int, layer: int):
        if self.dropout == 0.0 or layer == self.num_layers - 1:
            return x
        return drop(x, self.dropout, self.seed, call * self.num_layers + layer, step=self.mask_step)


class GRU(_LayerDropout):
    def __init__(self, input_size: int, hidden_size: int, num_layers: int = 1, bidirectional: bool = False,
                 batch_first: bool = False, device="cuda", generator=None, dropout: float = 0.0, seed: int = 0):
        import torch
        self._init_dropout(dropout, seed)
        self.input_size, self.hidden_size = input_size, hidden_size
        self.num_layers, self.bidirectional, self.batch_first = num_layers, bidirectional, batch_first
        dirs = 2 if bidirectional else 1
        self.params = {}
        k = hidden_size ** -0.5
        for l in range(num_layers):
            in_sz = input_size if l == 0 else hidden_size * dirs
            for sfx in ([""] + (["_reverse"] if bidirectional else [])):
                shapes = {f"weight_ih_l{l}{sfx}": (3 * hidden_size, in_sz),
                          f"weight_hh_l{l}{sfx}": (3 * hidden_size, hidden_size),
                          f"bias_ih_l{l}{sfx}": (3 * hidden_size,), f"bias_hh_l{l}{sfx}": (3 * hidden_size,)}
                for name, shp in shapes.items():
                    t = torch.empty(shp, dtype=torch.float32, device=device)
                    t.uniform_(-k, k, generator=generator)
                    self.params[name] = t

    def load_state_dict(self, state: dict) -> None:
        """Copy matching parameters (nn.js:58-80, Module.load_state_dict)."""
        for k, v in state.items():
            if k in self.params:
                if tuple(v.shape) != tuple(self.params[k].shape):
                    raise ValueError(f"{k}: shape {tuple(v.shape)} != {tuple(self.params[k].shape)}")
                self.params[k].copy_(v)

    def __call__(self, x, h0=None):
        return self.forward(x, h0)

    def forward(self, x, h0=None):
        import torch
        if self.batch_first:
            x = x.transpose(0, 1)
        x = x.contiguous()
        if x.dtype != torch.float32 or not x.is_cuda or x.dim() != 3:
            raise ValueError("x must be a 3-D float32 CUDA tensor")
        seq, batch = x.shape[0], x.shape[1]
        H, dirs = self.hidden_size, 2 if self.bidirectional else 1
        if h0 is not None:
            h0 = h0.contiguous()
            if tuple(h0.shape) != (self.num_layers * dirs, batch, H):
                raise ValueError("h0 must be [num_layers * num_directions, batch, hidden]")
        lib = _lib.load()
        stream = torch.cuda.current_stream().cuda_stream
        h_n = torch.empty((self.num_layers * dirs, batch, H), dtype=torch.float32, device=x.device)
        inp = x
        for l in range(self.num_layers):
            out = torch.empty((seq, batch, H * dirs), dtype=torch.float32, device=x.device)
            for d in range(dirs):
                sfx = "_reverse" if d else ""
                p = self.params
                h0p = h0[l * dirs + d].data_ptr() if h0 is not None else None
                _lib.check(lib.jst_gru_layer_forward(
                    inp.data_ptr(), seq, batch, inp.shape[2], H, p[f"weight_ih_l{l}{sfx}"].data_ptr(),
                    p[f"weight_hh_l{l}{sfx}"].data_ptr(), p[f"bias_ih_l{l}{sfx}"].data_ptr(),
                    p[f"bias_hh_l{l}{sfx}"].data_ptr(), h0p, d, out.data_ptr() + 4 * d * H, H * dirs,
                    h_n[l * dirs + d].data_ptr(), stream))
            inp = out
        if self.batch_first:
            inp = inp.transpose(0, 1)
        return inp, h_n

    # ------------------------------------------------------------ training
    def zero_grad(self) -> None:
        """Clear the accumulated parameter gradients (self.grads)."""
        for g in getattr(self, "grads", {}).values():
            g.zero_()

    def _check_x(self, x, h0):
        import torch
        if self.batch_first:
            x = x.transpose(0, 1)
        x = x.contiguous()
        if x.dtype != torch.float32 or not x.is_cuda or x.dim() != 3:
            raise ValueError("x must be a 3-D float32 CUDA tensor")
        dirs = 2 if self.bidirectional else 1
        if h0 is not None:
            h0 = h0.contiguous()
            if tuple(h0.shape) != (self.num_layers * dirs, x.shape[1], self.hidden_size):
                raise ValueError("h0 must be [num_layers * num_directions, batch, hidden]")
        return x, h0

    def forward_train(self, x, h0=None):
        """forward() that also keeps the gate values of every step for
        backward(); returns (output, h_n, ctx)."""
        import torch
        x, h0 = self._check_x(x, h0)
        seq, batch = x.shape[0], x.shape[1]
        H, dirs = self.hidden_size, 2 if self.bidirectional else 1
        lib = _lib.load()
        stream = torch.cuda.current_stream().cuda_stream
        h_n = torch.empty((self.num_layers * dirs, batch, H), dtype=torch.float32, device=x.device)
        call = self.calls
        inps, outs, saved = [], [], []
        inp = x
        for l in range(self.num_layers):
            out = torch.empty((seq, batch, H * dirs), dtype=torch.float32, device=x.device)
            sv = [torch.empty((seq, batch, 4 * H), dtype=torch.float32, device=x.device) for _ in range(dirs)]
            for d in range(dirs):
                sfx = "_reverse" if d else ""
                p = self.params
                h0p = h0[l * dirs + d].data_ptr() if h0 is not None else None
                _lib.check(lib.jst_gru_layer_forward_train(
                    inp.data_ptr(), seq, batch, inp.shape[2], H, p[f"weight_ih_l{l}{sfx}"].data_ptr(),
                    p[f"weight_hh_l{l}{sfx}"].data_ptr(), p[f"bias_ih_l{l}{sfx}"].data_ptr(),
                    p[f"bias_hh_l{l}{sfx}"].data_ptr(), h0p, d, out.data_ptr() + 4 * d * H, H * dirs,
                    h_n[l * dirs + d].data_ptr(), sv[d].data_ptr(), stream))
            inps.append(inp)
            outs.append(out)
            saved.append(sv)
            inp = self._drop(out, call, l)
        ctx = _TrainContext(seq, batch, inps, outs, saved, h0, call)
        self.calls += 1  # a refused call takes no masks
        output = inp.transpose(0, 1) if self.batch_first else inp
        return output, h_n, ctx

    def backward(self, ctx, dout, dh_n=None):
        """Back-propagate dL/d(output) (and dL/d(h_n)) through the pass of
        forward_train that produced ctx.  Adds every parameter's gradient to
        self.grads[name]; returns (dx, dh0) (dh0 None when no h0 was given)."""
        import torch
        if not hasattr(self, "grads"):
            self.grads = {k: torch.zeros_like(v) for k, v in self.params.items()}
        if self.batch_first:
            dout = dout.transpose(0, 1)
        g = dout.contiguous()
        seq, batch = ctx.seq, ctx.batch
        H, dirs = self.hidden_size, 2 if self.bidirectional else 1
        if tuple(g.shape) != (seq, batch, H * dirs):
            raise ValueError("dout must have the output's shape")
        if dh_n is not None:
            dh_n = dh_n.contiguous()
        lib = _lib.load()
        stream = torch.cuda.current_stream().cuda_stream
        dh0 = torch.empty_like(ctx.h0) if ctx.h0 is not None else None
        for l in range(self.num_layers - 1, -1, -1):
            inp, out = ctx.inps[l], ctx.outs[l]
            dinp = torch.empty_like(inp)
            for d in range(dirs):
                sfx = "_reverse" if d else ""
                p, gr = self.params, self.grads
                k = l * dirs + d
                acc = ACC_PARAMS | (ACC_DX if d else 0)
                _lib.check(lib.jst_gru_layer_backward(
                    inp.data_ptr(), seq, batch, inp.shape[2], H, p[f"weight_ih_l{l}{sfx}"].data_ptr(),
                    p[f"weight_hh_l{l}{sfx}"].data_ptr(), ctx.h0[k].data_ptr() if ctx.h0 is not None else None, d,
                    out.data_ptr() + 4 * d * H, H * dirs, ctx.saved[l][d].data_ptr(), g.data_ptr() + 4 * d * H,
                    H * dirs, dh_n[k].data_ptr() if dh_n is not None else None, dinp.data_ptr(),
                    gr[f"weight_ih_l{l}{sfx}"].data_ptr(), gr[f"weight_hh_l{l}{sfx}"].data_ptr(),
                    gr[f"bias_ih_l{l}{sfx}"].data_ptr(), gr[f"bias_hh_l{l}{sfx}"].data_ptr(),
                    dh0[k].data_ptr() if dh0 is not None else None, acc, stream))
            g = self._drop(dinp, ctx.call, l - 1) if l else dinp
        dx = g.transpose(0, 1) if self.batch_first else g
        return dx, dh0


# ------------------------------------------------------------ gated linear recurrence
CANDIDATES = {"tanh": 0, "identity": 1}  # JST_SCAN_* (include/jstorch_scan.h)


def _candidate(name: str) -> int:
    if name not in CANDIDATES:
        raise ValueError(f"candidate must be one of {sorted(CANDIDATES)} (got {name!r})")
    return CANDIDATES[name]


def gated_scan(gates, h0=None, *, lengths=None, reverse: bool = False, candidate: str = "tanh", out=None, h_n=None,
               stream=None):
    """(out, h_n) of h_t = z_t * h_{t-1} + (1 - z_t) * n_t over the steps of each sequence.

    gates: [seq, batch, 2 * hidden] float32, rows a | c (one pitch between all
    rows is allowed): z = sigmoid(a), n = tanh(c) ("tanh") or c ("identity").
    h0: [batch, hidden] (zeros when None).  lengths: int32 [batch] on the
    device; a sequence has its first lengths[b] steps (clamped to [0, seq]),
    behind them gates are not read and out is 0, and the state passes on.
    reverse runs each sequence from its last step to its first.  out [seq,
    batch, hidden] may have a pitch; h_n [batch, hidden] may be h0 itself.
    Runs asynchronously on `stream` (default: torch's current stream).
    """
    return _lib.calls().scan_forward(gates, h0, lengths, reverse, _candidate(candidate), out, h_n, stream)


def gated_scan_backward(gates, out, dout, h0=None, *, dh_n=None, lengths=None, reverse: bool = False,
                        candidate: str = "tanh", dgates=None, stream=None):
    """(dgates, dh0) of a gated_scan call: gates, h0, lengths, reverse and
    candidate as given to it, out as it returned it, dout = dL/dout and dh_n =
    dL/dh_n (either may be None: zero).  dgates is [seq, batch, 2 * hidden], 0
    behind a sequence's end; dh0 is None when h0 is.
    """
    return _lib.calls().scan_backward(gates, out, dout, h0, dh_n, lengths, reverse, _candidate(candidate), dgates, stream)


class GatedRNN(_LayerDropout):
    """Stacked gated linear recurrences: per layer and direction one projection
    gates = x . weight^T + bias (a GEMM over all steps) and gated_scan of them.

    Parameters weight_l{l}[_reverse] [2H, in] and bias_l{l}[_reverse] [2H], rows
    (a | c).  x [seq, batch, in] (or [batch, seq, in] with batch_first), h0
    [num_layers * directions, batch, H], lengths int32 [batch] as in gated_scan:
    what x and dout hold behind a sequence reaches no result.
    """

    def __init__(self, input_size: int, hidden_size: int, num_layers: int = 1, bidirectional: bool = False,
                 batch_first: bool = False, candidate: str = "tanh", device="cuda", generator=None,
                 dropout: float = 0.0, seed: int = 0):
        import torch
        _candidate(candidate)  # refuses other names
        self._init_dropout(dropout, seed)
        self.input_size, self.hidden_size, self.num_layers = input_size, hidden_size, num_layers
        self.bidirectional, self.batch_first, self.candidate = bidirectional, batch_first, candidate
        self.params, self.grads, self.quantized = {}, {}, None
        for l in range(num_layers):
            in_sz = input_size if l == 0 else hidden_size * (2 if bidirectional else 1)
            k = max(in_sz, 1) ** -0.5
            for sfx in self._suffixes():
                for name, shp in ((f"weight_l{l}{sfx}", (2 * hidden_size, in_sz)), (f"bias_l{l}{sfx}", (2 * hidden_size,))):
                    t = torch.empty(shp, dtype=torch.float32, device=device)
                    self.params[name] = t.uniform_(-k, k, generator=generator)

    def _suffixes(self):
        return ("", "_reverse") if self.bidirectional else ("",)

    def load_state_dict(self, state: dict) -> None:
        """Copy matching parameters; quantised weights are made again."""
        for k, v in state.items():
            if k in self.params:
                if tuple(v.shape) != tuple(self.params[k].shape):
                    raise ValueError(f"{k}: shape {tuple(v.shape)} != {tuple(self.params[k].shape)}")
                self.params[k].copy_(v)
        if self.quantized is not None:
            self.quantize()

    def quantize(self) -> "GatedRNN":
        """Run forward() and step() on 8-bit weights (quantize_rows of the
        present ones, one scale a channel) and 8-bit rows of the input, one
        scale a token.  Training keeps the float32 weights; call again after
        they change."""
        from .quant import quantize_rows
        self.quantized = {k: quantize_rows(v) for k, v in self.params.items() if k.startswith("weight")}
        return self

    def _project(self, x, l: int, sfx: str, serving: bool):
        """x [..., in] -> gates [..., 2H] of layer l."""
        w, b = f"weight_l{l}{sfx}", self.params[f"bias_l{l}{sfx}"]
        rows = x.reshape(x.shape[:-1].numel(), x.shape[-1])  # without a feature too
        if serving and self.quantized is not None:
            from .quant import linear_i8
            gates = linear_i8(rows, *self.quantized[w], bias=b)
        else:
            gates = gemm(rows, self.params[w].t(), bias=b)
        return gates.view(*x.shape[:-1], 2 * self.hidden_size)

    def _run(self, x, h0, lengths, train: bool):
        import torch
        if self.batch_first:
            x = x.transpose(0, 1)
        _lib.require_f32(x, "x")
        if x.dim() != 3 or x.shape[2] != self.input_size:
            raise ValueError(f"x must be [seq, batch, {self.input_size}]")
        x = x.contiguous()
        seq, batch, H, dirs = x.shape[0], x.shape[1], self.hidden_size, len(self._suffixes())
        if train and lengths is not None:  # rows behind a sequence meet dgates of 0 in the weights' gradient
            if not isinstance(lengths, torch.Tensor):
                raise TypeError("lengths must be a torch.Tensor")
            if lengths.shape != (batch,) or lengths.device != x.device:
                raise ValueError(f"lengths must be a contiguous int32 tensor of shape {(batch,)} on {x.device}")
            behind = torch.arange(seq, device=x.device)[:, None] >= lengths
            x = x.masked_fill(behind[..., None], 0.0)
        if h0 is not None and (tuple(h0.shape) != (self.num_layers * dirs, batch, H) or not h0.is_contiguous()):
            raise ValueError("h0 must be a contiguous [num_layers * num_directions, batch, hidden]")
        h_n = torch.empty((self.num_layers * dirs, batch, H), dtype=torch.float32, device=x.device)
        call = self.calls
        inps, outs, saved, inp = [], [], [], x
        for l in range(self.num_layers):
            out = torch.empty((seq, batch, H * dirs), dtype=torch.float32, device=x.device)
            kept = []
            for d, sfx in enumerate(self._suffixes()):
                gates = self._project(inp, l, sfx, not train)
                gated_scan(gates, h0[l * dirs + d] if h0 is not None else None, lengths=lengths, reverse=d == 1,
                           candidate=self.candidate, out=out[..., d * H:(d + 1) * H], h_n=h_n[l * dirs + d])
                kept.append(gates)
            if train:
                inps.append(inp)
                outs.append(out)
                saved.append(kept)
            inp = self._drop(out, call, l) if train else out
        ctx = _TrainContext(seq, batch, inps, outs, saved, h0, call) if train else None
        if train:
            ctx.lengths = lengths
            self.calls += 1  # a refused call takes no masks
        return inp.transpose(0, 1) if self.batch_first else inp, h_n, ctx

    def __call__(self, x, h0=None, lengths=None):
        return self.forward(x, h0, lengths)

    def forward(self, x, h0=None, lengths=None):
        return self._run(x, h0, lengths, False)[:2]

    def step(self, x, h):
        """One time step for serving: x [batch, in], h [num_layers, batch, H],
        updated in place; returns the last layer's new state (a view of h)."""
        if self.bidirectional:
            raise ValueError("step() needs a unidirectional model")
        _lib.require_f32(x, "x")
        if x.dim() != 2 or x.shape[1] != self.input_size:
            raise ValueError(f"x must be [batch, {self.input_size}]")
        if tuple(h.shape) != (self.num_layers, x.shape[0], self.hidden_size) or not h.is_contiguous():
            raise ValueError("h must be a contiguous [num_layers, batch, hidden]")
        for l in range(self.num_layers):
            gated_scan(self._project(x, l, "", True)[None], h[l], candidate=self.candidate, h_n=h[l])
            x = h[l]
        return x

    # ------------------------------------------------------------ training
    def zero_grad(self) -> None:
        """Clear the accumulated parameter gradients (self.grads)."""
        for g in self.grads.values():
            g.zero_()

    def forward_train(self, x, h0=None, lengths=None):
        """forward() on the float32 weights, with dropout, that also keeps what
        backward() needs; returns (output, h_n, ctx)."""
        return self._run(x, h0, lengths, True)

    def backward(self, ctx, dout, dh_n=None):
        """Back-propagate dL/d(output) (and dL/d(h_n)) through the pass that
        made ctx.  Adds every parameter's gradient to self.grads[name]; returns
        (dx, dh0) (dh0 None when no h0 was given)."""
        import torch
        if not self.grads:
            self.grads = {k: torch.zeros_like(v) for k, v in self.params.items()}
        g = (dout.transpose(0, 1) if self.batch_first else dout).contiguous()
        H, dirs, rows = self.hidden_size, len(self._suffixes()), ctx.seq * ctx.batch
        if tuple(g.shape) != (ctx.seq, ctx.batch, H * dirs):
            raise ValueError("dout must have the output's shape")
        if dh_n is not None:
            dh_n = dh_n.contiguous()
        dh0 = torch.empty_like(ctx.h0) if ctx.h0 is not None else None
        ones = torch.ones((1, rows), dtype=torch.float32, device=g.device)
        for l in range(self.num_layers - 1, -1, -1):
            inp, dinp = ctx.inps[l].view(rows, ctx.inps[l].shape[2]), None
            for d, sfx in enumerate(self._suffixes()):
                k, cols = l * dirs + d, slice(d * H, (d + 1) * H)
                dgates, dh = gated_scan_backward(
                    ctx.saved[l][d], ctx.outs[l][..., cols], g[..., cols], ctx.h0[k] if ctx.h0 is not None else None,
                    dh_n=dh_n[k] if dh_n is not None else None, lengths=ctx.lengths, reverse=d == 1,
                    candidate=self.candidate)
                if dh0 is not None:
                    dh0[k] = dh
                dg = dgates.view(rows, 2 * H)
                self.grads[f"weight_l{l}{sfx}"] += gemm(dg.t(), inp)
                self.grads[f"bias_l{l}{sfx}"] += gemm(ones, dg)[0]
                dx = gemm(dg, self.params[f"weight_l{l}{sfx}"])
                dinp = dx if dinp is None else dinp.add_(dx)
            g = dinp.view(ctx.seq, ctx.batch, inp.shape[1])
            if l:
                g = self._drop(g, ctx.call, l - 1)
        return g.transpose(0, 1) if self.batch_first else g, dh0
