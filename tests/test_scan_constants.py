"""The constants of csrc/scan.cu's exponential and tanh, read from the source and held to what its comments say."""
import re
from pathlib import Path

import numpy as np

SOURCE = (Path(__file__).parents[1] / "jstorch_b200/csrc/scan.cu").read_text()


def _floats(text):
    return [float(np.float32(v)) for v in re.findall(r"(-?\d+\.\d+(?:e-\d+)?)f", text)]


def _tanh_coefficients():
    body = SOURCE[SOURCE.index("const F<V> q = c * c;"):SOURCE.index("const F<V> near =")]
    top, *rest = _floats(body)
    return np.array([top, *rest])[::-1]  # of c^3, c^5, ...


def test_tanh_polynomial():
    """c + c^3 P(c^2) is within 0.08 of 2^-24 of tanh up to 0.6 (its evaluation rounds on top of that)."""
    c = np.linspace(1e-3, 0.6, 300001)
    p = _tanh_coefficients()
    assert len(p) == 5
    off = (c + c ** 3 * np.polyval(p[::-1], c * c)) / np.tanh(c) - 1
    assert np.abs(off).max() < 0.08 * 2.0 ** -24


def test_tanh_polynomial_is_the_minimax_one():
    """The coefficients are those of the smallest largest relative error, solved for as a linear programme over
    Chebyshev points of (0, 0.6] and rounded to fp32: found again to 2e-6 of each."""
    from scipy.optimize import linprog
    n = 2000
    x = 0.3 * (1 - np.cos(np.pi * (np.arange(n) + 0.5) / n))
    x = x[x > 1e-3]
    rows = x[:, None] ** (2 * np.arange(5) + 3) / np.tanh(x)[:, None] * 2.0 ** 24
    rest = (1 - x / np.tanh(x)) * 2.0 ** 24
    bound = -np.ones((len(x), 1))
    r = linprog(np.r_[np.zeros(5), 1.0], A_ub=np.block([[rows, bound], [-rows, bound]]), b_ub=np.concatenate([rest, -rest]),
                bounds=[(None, None)] * 6, method="highs-ds")
    assert r.status == 0 and r.x[5] < 0.05
    np.testing.assert_allclose(_tanh_coefficients(), r.x[:5], rtol=2e-6)


def test_split_constants():
    """log2 e as two fp32 numbers to 2^-48, and ln 2."""
    high, low = _floats(SOURCE[SOURCE.index("const float log2e = TIMES"):SOURCE.index("const F<V> t = x * all<V>(-log2e)")])
    assert abs(high + low - np.log2(np.e)) < 2.0 ** -48
    (ln2,) = _floats(re.search(r"-log2e_rest\), r\) \* all<V>\(([^)]*)\)", SOURCE)[1])
    assert ln2 == float(np.float32(np.log(2.0)))
