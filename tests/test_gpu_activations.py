"""The activations of the linear layer and their slopes where they can go wrong: far tails, values whose exponentials
leave fp32's range, infinities and NaN, against fp64 forms.  A bias that is added to a product of zeros hands the kernels
every value exactly as it is.

Tolerances count roundings, u = 2^-24 each: the chip's 2^x is good to an ulp (2 u), and the correction for what its
argument lost rounds once more; a reciprocal with a step of Newton's method is off by 2 u."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F = np.float32
U = 2.0 ** -24
LEAST = 2.0 ** -126   # the smallest normal number

_SIZES = [1e-20, 1e-3, 0.5, 1, 1.2784645, 2, 3, 5, 7, 10, 12, 12.9, 13.1, 13.3, 14, 19.9, 20.1, 30, 50, 79.9, 80.1, 83, 83.5, 84, 87, 88, 90,
          95, 100, 103, 104.5, 109, 111, 127, 129, 1e3, 1e10, 1e30, 2.3e38, 2.4e38, 3.4e38]
FINITE = np.array([0.0] + _SIZES + [-v for v in _SIZES], dtype=F)
SPREAD = np.random.RandomState(3).uniform(-115, 115, 400).astype(F)
Z = np.concatenate([FINITE, SPREAD])


def _erfc(z):
    return np.vectorize(math.erfc, otypes=[float])(z)


def _forward(cl, act, z):
    """act(z), and z as the layer kept it, by a small launch and by the tiled kernels"""
    got = []
    for rows in (3, 130):
        pre, y = cl.ClTensor(), cl.ClTensor()
        zeros = cl.ClTensor(np.zeros((rows, 4), dtype=F))
        y.linear(zeros, cl.ClTensor(np.zeros((z.size, 4), dtype=F)), cl.ClTensor(z), activation=act, preact=pre)
        kept, y = pre.float(), y.float()
        assert np.array_equal(kept[0], z, equal_nan=True)
        assert all(np.array_equal(y[r], y[0], equal_nan=True) for r in range(rows))
        got.append(y[0])
    assert np.array_equal(got[0], got[1], equal_nan=True)
    return got[0].astype(np.float64)


def _slope(cl, act, z):
    """act'(z): one row whose gradient is 1 leaves it in the bias gradient, and through a product with 1 in the weight's"""
    gw, gb = cl.ClTensor(), cl.ClTensor()
    one = cl.ClTensor(np.ones((1, 1), dtype=F))
    cl.linearBackward(None, gw, gb, cl.ClTensor(np.ones((1, z.size), dtype=F)), one, cl.ClTensor(np.ones((z.size, 1), dtype=F)),
                      preact=cl.ClTensor(z.reshape(1, -1)), activation=act)
    by_bias, by_weight = gb.float(), gw.float()[:, 0]
    # fp32 products may take numbers below the normal range to zero
    assert np.array_equal(np.where(np.abs(by_bias) < LEAST, 0, by_bias), np.where(np.abs(by_weight) < LEAST, 0, by_weight), equal_nan=True)
    return by_bias.astype(np.float64)


def _within(got, want, tol, z, what):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), [(float(a), float(b), float(c)) for a, b, c in zip(z[bad][:4], got[bad][:4], want[bad][:4])])


def _silu(z):
    with np.errstate(over="ignore"):
        return np.where(z >= 0, 1, 0) * z / (1 + np.exp(-np.abs(z))) + np.where(z < 0, z, 0) * np.exp(-np.abs(z)) / (1 + np.exp(-np.abs(z)))


def test_silu_of_far_values(cl):
    """exp 4 u, twice (numerator and denominator), the sum one, the reciprocal 2 u, three products"""
    z64 = Z.astype(np.float64)
    want = _silu(z64)
    _within(_forward(cl, "silu", Z), want, 14 * U * np.abs(want) + LEAST * U * 4, Z, "silu")


def test_slope_of_silu_of_far_values(cl):
    """s = sigmoid(z) and 1 - s are off by 12 u each, which z multiplies; two roundings of the sum and the product"""
    z64 = Z.astype(np.float64)
    e = np.exp(-np.abs(z64))
    s, rest = np.where(z64 >= 0, 1, e) / (1 + e), np.where(z64 >= 0, e, 1) / (1 + e)
    want = s * (1 + z64 * rest)
    _within(_slope(cl, "silu", Z), want, U * s * (14 + 26 * np.abs(z64) * rest) + LEAST, Z, "slope of silu")


def test_activations_of_what_is_not_finite(cl):
    z = np.array([np.inf, -np.inf, np.nan, 0.0, 1.0], dtype=F)
    for act in ("relu", "gelu", "silu"):
        y = _forward(cl, act, z)
        assert y[0] == np.inf and y[1] == 0 and np.isnan(y[2]) and y[3] == 0 and np.isfinite(y[4]), (act, y)
    for act in ("gelu", "silu"):
        s = _slope(cl, act, z)
        assert s[0] == 1 and s[1] == 0 and np.isnan(s[2]) and s[3] == 0.5 and np.isfinite(s[4]), (act, s)
    s = _slope(cl, "relu", z)
    assert s[0] == 1 and s[1] == 0 and s[3] == 0 and s[4] == 1


def _tails(z):
    """the normal distribution's mass beyond |z| on one side"""
    return 0.5 * _erfc(np.abs(z) / math.sqrt(2))


# The tail is t p(t) exp(-z^2 / 2) / 2 with t = 3 / (3 + |z| / sqrt 2).  t is off by 5 u (a product, a sum, a reciprocal,
# a product), which its polynomial passes on up to 3.4 times; the polynomial's own roundings come to 4 u, the
# exponential's to 4 u, the products' to 3 u: 28 u of the tail.
TAIL = 28 * U


def test_gelu_of_far_values(cl):
    z64 = Z.astype(np.float64)
    tail = np.abs(z64) * _tails(z64)
    want = np.maximum(z64, 0) - tail
    _within(_forward(cl, "gelu", Z), want, TAIL * tail + 2 * U * np.abs(want) + LEAST, Z, "gelu")


def test_slope_of_gelu_of_far_values(cl):
    """the density is off by the exponential's 4 u and two products"""
    z64 = Z.astype(np.float64)
    tail, density = _tails(z64), np.abs(z64) * np.exp(-z64 * z64 / 2) / math.sqrt(2 * math.pi)
    want = np.where(z64 > 0, 1 - tail + density, tail - density)
    _within(_slope(cl, "gelu", Z), want, TAIL * tail + 7 * U * density + 2 * U * np.abs(want) + 20 * LEAST, Z, "slope of gelu")
