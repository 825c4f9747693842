"""quantize_rows, gemm_i8 and linear_i8 where the definitions are sharp: the scale as a
quotient, scales whose product leaves the type, empty operands, outputs beside inputs."""
import numpy as np
import pytest

from oracle import oracle

pytestmark = pytest.mark.gpu


def _dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def test_scale_is_the_rounded_quotient():
    """max|x| / 127 to the nearest fp32 number (a product with the rounded 1 / 127 misses it for one peak in twenty),
    and q the nearest integer to x over it, for rows of either form of the kernels."""
    from jstorch_b200 import quant
    rng = np.random.default_rng(7)
    x = (rng.standard_normal((5000, 40)) * np.exp(rng.uniform(-60, 60, (5000, 1)))).astype(np.float32)
    peak = np.abs(x).max(axis=1).astype(np.float64)
    scale = (peak / 127).astype(np.float32)
    assert (scale != (peak.astype(np.float32) * np.float32(1 / 127))).mean() > 0.03
    want = np.rint(x.astype(np.float64) / scale.astype(np.float64)[:, None])
    q, s = quant.quantize_rows(_dev(x))
    np.testing.assert_array_equal(s.cpu().numpy(), scale)
    np.testing.assert_array_equal(q.cpu().numpy(), want)
    # the product's own quantisation: an identity weight shows q * scale, rows one by one and a few together
    one = np.ones(40, np.float32)
    for rows in (1, 8, 70):
        y = quant.linear_i8(_dev(x[:rows]), _dev(np.eye(40, dtype=np.int8)), _dev(one)).cpu().numpy()
        np.testing.assert_array_equal(y, want[:rows].astype(np.float32) * scale[:rows, None])


@pytest.mark.parametrize("M", [1, 5, 40, 100, 700])
def test_scales_whose_product_leaves_the_type(M):
    """A product of scales below 2^-126 or above 2^128 costs no digits, and no zero, of a result within the type."""
    from jstorch_b200 import quant
    rng = np.random.default_rng(M)
    N, K = 300, 512
    a, w = (rng.integers(-128, 128, (n, K), dtype=np.int8) for n in (M, N))
    a[::3] = 0  # sums of 0
    w[::5, 1:] = 0  # small sums
    for sa, sw in ((1e-30, 1e-9), (1e-9, 1e-30), (1e-42, 1e30), (1e30, 1e-42), (3e38, 1e-9), (1e-9, 3e38), (1e20, 1e20), (1e38, 1e38)):
        a_scale, w_scale = (np.full(n, s, np.float32) * rng.uniform(0.5, 1, n).astype(np.float32) for n, s in ((M, sa), (N, sw)))
        value, bound = oracle.gemm_i8_f64(a, w, a_scale, w_scale)
        for lay in (_dev(a), _dev(np.pad(a, ((0, 0), (0, 16))))[:, :K]):
            got = quant.gemm_i8(lay, _dev(w), _dev(a_scale), _dev(w_scale)).cpu().numpy().astype(np.float64)
            over = np.abs(value) >= 2.0 ** 128
            assert np.isinf(got[over]).all() and np.array_equal(np.sign(got[over]), np.sign(value[over]))
            assert (np.abs(got - value)[~over] <= bound[~over]).all(), (sa, sw)


@pytest.mark.parametrize("M,N", [(5, 0), (0, 3), (0, 0)])
def test_empty_products_with_a_bias(M, N):
    import torch
    from jstorch_b200 import quant
    w, s, b = torch.zeros((N, 16), dtype=torch.int8, device="cuda"), torch.ones(N, device="cuda"), torch.zeros(N, device="cuda")
    for relu in (False, True):
        assert quant.linear_i8(torch.zeros((M, 16), device="cuda"), w, s, bias=b, relu=relu).shape == (M, N)
        a = torch.zeros((M, 16), dtype=torch.int8, device="cuda")
        assert quant.gemm_i8(a, w, torch.ones(M, device="cuda"), s, bias=b, relu=relu).shape == (M, N)
