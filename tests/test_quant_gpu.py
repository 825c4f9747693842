"""quantize_rows, gemm_i8 and linear_i8 against the fp64 oracle: the quantised
values and scales are equal, the products within the four roundings that
oracle.gemm_i8_f64 counts."""
import numpy as np
import pytest

from oracle import oracle

pytestmark = pytest.mark.gpu


def _dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _held(got, want):
    value, bound = want
    got = got.cpu().numpy().astype(np.float64)
    assert got.shape == value.shape
    # from half a step above the largest fp32 number on, a value rounds to an infinity of its sign
    border = 2.0 ** 128 - 2.0 ** 103
    beyond, may = np.abs(value) - bound >= border, np.abs(value) + bound >= border
    assert np.array_equal(got[beyond], np.copysign(np.inf, value[beyond]))
    skip = beyond | (may & np.isinf(got) & (np.sign(got) == np.sign(value)))
    off = np.where(skip, 0.0, np.abs(np.where(skip, 0.0, got) - np.where(skip, 0.0, value)))
    assert np.all(off <= bound), (float(np.max(off - bound)), np.unravel_index(np.argmax(off - bound), off.shape))


def _operands(M, N, K, seed=0):
    rng = np.random.default_rng([seed, M, N, K])
    a = rng.integers(-128, 128, (M, K), dtype=np.int8)
    w = rng.integers(-128, 128, (N, K), dtype=np.int8)
    return (a, w, rng.uniform(1e-3, 2.0, M).astype(np.float32), rng.uniform(1e-3, 2.0, N).astype(np.float32),
            (rng.standard_normal(N) * 1e4).astype(np.float32))


def _aligned(x):
    """Rows at multiples of 16 bytes, as quantize_rows lays them out."""
    import torch
    rows, cols = x.shape
    held = torch.full((rows, max((cols + 15) // 16 * 16, 16)), 99, dtype=torch.int8, device="cuda")  # not zeros
    held[:, :cols] = _dev(x)
    return held[:, :cols]


SIZES = [(1, 1, 1), (1, 7, 3), (1, 128, 64), (1, 1000, 4096), (1, 20, 1024), (1, 21, 1025), (1, 40, 8192), (1, 33, 8195),
         (1, 50, 20001), (1, 1024, 8208), (65, 1, 8191), (130, 257, 8000), (999, 65, 7000), (200, 2048, 4096), (1, 1301, 20000), (2, 1, 5), (6, 3000, 700), (16, 5, 640), (40, 130, 2050), (64, 1500, 129), (65, 300, 40), (2, 33, 100), (3, 64, 16), (4, 129, 515), (5, 256, 512),
         (7, 31, 77), (8, 512, 1024), (9, 100, 260), (15, 65, 48), (16, 130, 1000), (17, 64, 128), (31, 200, 96),
         (33, 257, 129), (64, 64, 64), (100, 300, 1031), (127, 128, 127), (128, 256, 128), (129, 257, 144),
         (200, 513, 2000), (256, 1024, 784), (300, 70, 6000), (513, 129, 17), (1000, 5, 300)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("aligned", [True, False])
def test_product(M, N, K, aligned):
    from jstorch_b200 import quant
    a, w, sa, sw, b = _operands(M, N, K)
    lay = _aligned if aligned else _dev
    _held(quant.gemm_i8(lay(a), lay(w), _dev(sa), _dev(sw)), oracle.gemm_i8_f64(a, w, sa, sw))
    _held(quant.gemm_i8(lay(a), lay(w), _dev(sa), _dev(sw), bias=_dev(b), relu=True),
          oracle.gemm_i8_f64(a, w, sa, sw, b, True))


@pytest.mark.parametrize("M,N,K", [(600, 9000, 300), (2400, 2600, 1000), (4000, 4100, 200), (700, 4096, 128)])
def test_many_tiles(M, N, K):
    """Several tiles a processor, in each of the kernel's tile forms; C with and without 16-byte rows."""
    import torch
    from jstorch_b200 import quant
    a, w, sa, sw, b = _operands(M, N, K)
    want = torch.from_numpy(a).cuda().double() @ torch.from_numpy(w).cuda().double().t()
    scale = _dev(sa).double()[:, None] * _dev(sw).double()
    # oracle.gemm_i8_f64 on the device: three roundings of the product, one of the sum
    value = want * scale + _dev(b).double()
    bound = 2.0 ** -24 * (3.001 * (want * scale).abs() + value.abs()) * 1.001 + (want.abs() + 1) * 2.0 ** -150
    for gap in (0, 1):
        held = torch.full((M, N + gap), 7.0, device="cuda")
        quant.gemm_i8(_aligned(a), _aligned(w), _dev(sa), _dev(sw), out=held[:, :N], bias=_dev(b))
        assert bool(((held[:, :N].double() - value).abs() <= bound).all())
        assert bool((held[:, N:] == 7).all())


@pytest.mark.parametrize("M,N,K", [(70000, 33000, 16), (300000, 16, 8192), (1, 300000, 8192)])
def test_offsets_past_32_bits(M, N, K):
    """Outputs of more than 2^31 values, operands of more than 2^31 bytes: the last rows and columns are right."""
    import torch
    from jstorch_b200 import quant
    g = torch.Generator(device="cuda").manual_seed(M)
    a, w = (torch.randint(-128, 128, (n, K), generator=g, device="cuda", dtype=torch.int8) for n in (M, N))
    sa, sw = (torch.rand(n, generator=g, device="cuda") + 0.5 for n in (M, N))
    y = quant.gemm_i8(a, w, sa, sw)
    m, n = min(M, 40), min(N, 40)
    want = oracle.gemm_i8_f64(a[-m:].cpu().numpy(), w[-n:].cpu().numpy(), sa[-m:].cpu().numpy(), sw[-n:].cpu().numpy())
    _held(y[-m:, -n:], want)
    del y, a
    if M > 1000 and K > 1000:
        x = torch.randn((M, K), generator=g, device="cuda")
        q, s = quant.quantize_rows(x)
        want_q, want_s = oracle.quantize_rows(x[-5:].cpu().numpy())
        assert np.array_equal(q[-5:].cpu().numpy(), want_q) and np.array_equal(s[-5:].cpu().numpy(), want_s)


@pytest.mark.parametrize("M,N,K", [(1, 5, 131071), (9, 70, 131071), (130, 130, 131071)])
def test_largest_sums(M, N, K):
    """-128 * -128 summed over the longest row: 2^31 - 2^14 fits 32 bits."""
    import torch
    from jstorch_b200 import quant
    a = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    w = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    one = [torch.ones(n, device="cuda") for n in (M, N)]
    y = quant.gemm_i8(a, w, *one)
    assert bool((y == float(np.float32(16384.0 * K))).all())


def test_empty_and_zero_length():
    import torch
    from jstorch_b200 import quant
    for M, N in ((0, 5), (5, 0)):
        y = quant.gemm_i8(*(torch.zeros((n, 16), dtype=torch.int8, device="cuda") for n in (M, N)),
                          torch.ones(M, device="cuda"), torch.ones(N, device="cuda"))
        assert y.shape == (M, N)
    b = torch.tensor([1.0, -2.0, 3.0], device="cuda")
    for m in (2, 200):
        args = (torch.zeros((m, 0), dtype=torch.int8, device="cuda"), torch.zeros((3, 0), dtype=torch.int8, device="cuda"),
                torch.ones(m, device="cuda"), torch.ones(3, device="cuda"))
        assert quant.gemm_i8(*args, bias=b, relu=True).tolist() == [[1.0, 0.0, 3.0]] * m
        y = quant.linear_i8(torch.zeros((m, 0), device="cuda"), args[1], args[3], bias=b)
        assert y.tolist() == [[1.0, -2.0, 3.0]] * m
    assert quant.linear_i8(torch.zeros((0, 4), device="cuda"), torch.zeros((3, 4), dtype=torch.int8, device="cuda"),
                           torch.ones(3, device="cuda")).shape == (0, 3)


@pytest.mark.parametrize("M", [1, 6, 40, 200])
def test_output_pitch_leaves_gaps_alone(M):
    import torch
    from jstorch_b200 import quant
    for N, gap in ((70, 3), (256, 4), (261, 1)):
        a, w, sa, sw, b = _operands(M, N, 90)
        held = torch.full((M + 2, N + gap), 7.0, device="cuda")
        quant.gemm_i8(_aligned(a), _aligned(w), _dev(sa), _dev(sw), out=held[1:M + 1, :N], bias=_dev(b))
        _held(held[1:M + 1, :N], oracle.gemm_i8_f64(a, w, sa, sw, b))
        assert bool((held[0] == 7).all()) and bool((held[M + 1] == 7).all()) and bool((held[:, N:] == 7).all())


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (2, 16), (5, 255), (4, 256), (7, 1000), (2, 4097), (33, 8192),
                                       (1, 20000), (3, 40001), (1200, 1),
                                       (1500, 100), (1203, 1021), (1184, 1024), (1300, 1025)])
def test_quantize_rows(rows, cols):
    from jstorch_b200 import quant
    rng = np.random.default_rng([rows, cols])
    x = (rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal((rows, 1)) * 4)).astype(np.float32)
    q, s = quant.quantize_rows(_dev(x))
    want_q, want_s = oracle.quantize_rows(x)
    np.testing.assert_array_equal(s.cpu().numpy(), want_s)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    assert q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0


def _hard_rows(cols):
    """Halves, their neighbours, denormals, extremes, zeros, and rows that are not finite."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((12, cols)).astype(np.float32)
    for r, s in ((0, 1.0), (1, 0.37), (2, 3.3e-5)):  # quotients at and next to a half
        s = np.float32(s)
        half = ((rng.integers(-127, 127, cols) + 0.5) * np.float64(s)).astype(np.float32)
        x[r] = np.nextafter(half, np.where(rng.random(cols) < 0.5, np.inf, -np.inf).astype(np.float32))
        x[r, ::3] = half[::3]
        x[r, 0] = 127 * s
    x[3] *= np.float32(1e-44)
    x[4] = np.float32(1e-45)
    x[5] = 0.0
    x[6] *= np.float32(3e37)
    x[7, cols // 2], x[8, cols - 1], x[9, 0] = np.inf, -np.inf, np.nan
    x[10] *= np.float32(1e-38)
    x[11] = -0.0
    return x


@pytest.mark.parametrize("cols", [64, 257, 4096])
def test_quantize_hard_rows(cols):
    from jstorch_b200 import quant
    x = _hard_rows(cols)
    q, s = quant.quantize_rows(_dev(x))
    want_q, want_s = oracle.quantize_rows(x)
    np.testing.assert_array_equal(s.cpu().numpy(), want_s)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)


def test_quantize_borders():
    """Every half within the range, and the numbers up to three steps around it, at scales of every size."""
    from jstorch_b200 import quant
    rng = np.random.default_rng(3)
    scales = np.exp(rng.uniform(np.log(1e-37), np.log(1e36), 300)).astype(np.float32)
    scales = np.concatenate([scales, np.float32(2.0) ** np.arange(-104, -96, dtype=np.float32), np.float32([1.0, 0.75])])
    halves = np.arange(-126.5, 127.0)
    x = (halves[None, :, None] * scales.astype(np.float64)[:, None, None]).astype(np.float32)
    x = np.repeat(x, 7, axis=2)
    for k in range(7):
        for _ in range(abs(k - 3)):
            x[..., k] = np.nextafter(x[..., k], np.float32(np.inf if k > 3 else -np.inf))
    x = x.reshape(len(scales), -1)
    x[:, 0] = np.float32(127.0) * scales
    q, s = quant.quantize_rows(_dev(x))
    want_q, want_s = oracle.quantize_rows(x)
    np.testing.assert_array_equal(s.cpu().numpy(), want_s)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)


@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear(M, N, K):
    from jstorch_b200 import quant
    rng = np.random.default_rng([9, M, N, K])
    x = (rng.standard_normal((M, K)) * np.exp(rng.standard_normal((M, 1)))).astype(np.float32)
    _, w, _, sw, b = _operands(M, N, K)
    q, s = oracle.quantize_rows(x)
    y = quant.linear_i8(_dev(x), _aligned(w), _dev(sw), bias=_dev(b))
    _held(y, oracle.gemm_i8_f64(q, w, s, sw, b))
    # the two calls that it stands for, bit for bit
    qd, sd = quant.quantize_rows(_dev(x))
    assert np.array_equal(y.cpu().numpy(), quant.gemm_i8(qd, _aligned(w), sd, _dev(sw), bias=_dev(b)).cpu().numpy())
    # rows with a pitch, a weight without alignment
    held = _dev(np.concatenate([x, x[:, :1] + 9], axis=1))
    want = oracle.gemm_i8_f64(q, w, s, sw, b, True)
    _held(quant.linear_i8(held[:, :K], _dev(w), _dev(sw), bias=_dev(b), relu=True), want)
    _held(quant.linear_i8(held[:, :K], _aligned(w), _dev(sw), bias=_dev(b), relu=True), want)


@pytest.mark.parametrize("repeat", [1, 20])
def test_linear_hard_rows(repeat):
    """Few rows and many: the same values, and a row that is not finite is NaN throughout, alone."""
    import torch
    from jstorch_b200 import quant
    x = np.tile(_hard_rows(272), (repeat, 1))
    _, w, _, sw, _ = _operands(len(x), 150, 272)
    y = quant.linear_i8(_dev(x), _aligned(w), _dev(sw))
    q, s = oracle.quantize_rows(x)
    fine = np.isfinite(s)
    value, bound = oracle.gemm_i8_f64(q[fine], w, s[fine], sw)
    _held(y[torch.from_numpy(fine)], (value, bound))
    assert bool(torch.isnan(y[torch.from_numpy(~fine)]).all())
    if repeat == 1:
        for r in range(len(x)):  # one row at a time: the form for single tokens
            one = quant.linear_i8(_dev(x[r:r + 1]), _aligned(w), _dev(sw))
            assert np.array_equal(one.cpu().numpy(), y[r:r + 1].cpu().numpy(), equal_nan=True)


def test_another_stream_and_captured_graphs():
    """Two graphs captured before either runs, replayed in turn and on two streams at once."""
    import torch
    from jstorch_b200 import quant
    rng = np.random.default_rng(1)
    sizes = [(1, 300, 500), (6, 64, 1000), (300, 270, 500)]
    work = []
    for M, N, K in sizes:
        x = rng.standard_normal((M, K)).astype(np.float32)
        _, w, _, sw, _ = _operands(M, N, K)
        work.append((_dev(x), _dev(w), _dev(sw)))  # rows of no alignment: workspaces too
    want = [quant.linear_i8(*c) for c in work]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = [quant.linear_i8(*c, stream=side) for c in work]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for c in work:
        held, g = torch.zeros_like(c[0]), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = quant.linear_i8(held, *c[1:])
        graphs.append((g, held, y))
    for _ in range(3):
        for (g, held, y), c in zip(graphs, work):
            held.copy_(c[0])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (g, held, y), ref in zip(graphs, want):
            assert torch.equal(y, ref)
            held.zero_()


def test_threads_on_their_own_streams():
    """Several host threads at once: the entry points keep nothing of one call for another."""
    import threading

    import torch
    from jstorch_b200 import quant
    sizes = [(1, 300, 500), (6, 64, 1000), (100, 270, 515), (1000, 1000, 512)]
    cases, want = [], []
    for M, N, K in sizes:
        x = np.random.default_rng(M).standard_normal((M, K)).astype(np.float32)
        _, w, _, sw, _ = _operands(M, N, K)
        cases.append((_dev(x), _dev(w), _dev(sw)))
        want.append(quant.linear_i8(*cases[-1]))
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for k in range(20):
                c = (i + k) % len(cases)
                y = quant.linear_i8(*cases[c])
                s.synchronize()
                if not torch.equal(y, want[c]):
                    bad.append((i, c))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_repeats_bit_for_bit_and_keeps_its_inputs():
    import torch
    from jstorch_b200 import quant
    for M, N, K in ((5, 300, 515), (700, 700, 700)):
        a, w, sa, sw, b = _operands(M, N, K)
        held = [_dev(v) for v in (a, w, sa, sw, b)]
        first = quant.gemm_i8(*held[:4], bias=held[4])
        assert torch.equal(first, quant.gemm_i8(*held[:4], bias=held[4]))
        assert all(np.array_equal(h.cpu().numpy(), v) for h, v in zip(held, (a, w, sa, sw, b)))
    import jstorch_b200
    assert jstorch_b200.device_error() == 0


def test_refusals():
    import torch
    from jstorch_b200 import quant
    q, x = torch.zeros((4, 16), dtype=torch.int8, device="cuda"), torch.zeros((4, 16), device="cuda")
    s = torch.ones(4, device="cuda")
    bad = [
        lambda: quant.gemm_i8(q, q[:, :8], s, s), lambda: quant.gemm_i8(q.t(), q.t(), s, s),
        lambda: quant.gemm_i8(q[0], q, s, s), lambda: quant.gemm_i8(q, q, s[:3], s), lambda: quant.gemm_i8(q, q, s, s[::2]),
        lambda: quant.gemm_i8(q, q, s, s, bias=s[:2]), lambda: quant.gemm_i8(q, q, s, s, out=x),
        lambda: quant.gemm_i8(q, q, s, s, out=torch.zeros((4, 4), device="cuda").t()),
        lambda: quant.gemm_i8(q, q, s.cpu(), s), lambda: quant.linear_i8(x[:, :8], q, s), lambda: quant.linear_i8(x.t(), q, s),
        lambda: quant.linear_i8(x, q, s.cpu()), lambda: quant.quantize_rows(x[0]), lambda: quant.quantize_rows(x.t()),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        quant.gemm_i8(q.to(torch.uint8), q, s, s)
    with pytest.raises(TypeError):
        quant.linear_i8(x.half(), q, s)


def test_sizes_past_32_bits_are_refused():
    """The C entry points count rows in 32 bits: a larger tensor must not wrap to a smaller one."""
    import torch
    from jstorch_b200 import quant
    rows = torch.zeros((2 ** 32 + 4, 0), device="cuda")
    q = rows.to(torch.int8)
    one = torch.ones(3, device="cuda")
    for call in (lambda: quant.quantize_rows(rows), lambda: quant.linear_i8(rows, q[:3], one),
                 lambda: quant.linear_i8(rows[:3], q, one), lambda: quant.gemm_i8(q[:3], q, one, one)):
        with pytest.raises(ValueError, match="size >"):
            call()
