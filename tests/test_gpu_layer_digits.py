"""The products of the layer operators keep all 24 bits of their operands in every tile: whole results are held to the
error that fp32 sums have in the norm.

A running sum of K products of independent entries of random sign has size sqrt(j) after j of them, each addition rounds
it by 0.58 u rms, u = 2^-24, which makes 0.41 sqrt(K) u of the result's norm.  Twice that is allowed; 16 keeps short sums
from being held to less than a few roundings.  Operands cut to 16 bits would be off by some 2^-18, which is more than that
up to K = 5000."""
import math
import zlib

import numpy as np
import pytest

from layer_shapes import GROUPED, LINEAR

F = np.float32
U = 2.0 ** -24


def _rng(*key):
    return np.random.RandomState(zlib.crc32(repr(key).encode()) & 0x7FFFFFFF)


def _normal(rng, *shape):
    return rng.standard_normal(shape).astype(F)


def _error(got, want):
    return np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want)


def _allowed(depth):
    return 0.82 * math.sqrt(max(depth, 16)) * U


def _check(got, a, b, what):
    want = a.astype(np.float64) @ b.astype(np.float64)
    assert _error(got, want) <= _allowed(a.shape[1]), (what, _error(got, want), _allowed(a.shape[1]))


def _parts(x, n):
    """the sum of n bf16 values nearest to x"""
    out, rest = np.zeros(x.shape), x.astype(np.float64)
    for _ in range(n):
        bits = rest.astype(F).view(np.uint32)
        part = ((bits + 0x7FFF + ((bits >> 16) & 1)) & np.uint32(0xFFFF0000)).view(F).astype(np.float64)
        out, rest = out + part, rest - part
    return out


@pytest.mark.parametrize("depth", [40, 300, 1030, 4100])
def test_the_bound_sees_operands_of_16_bits(depth):
    g = _rng("parts", depth)
    a, b = _normal(g, 64, depth), _normal(g, depth, 64)
    want = a.astype(np.float64) @ b.astype(np.float64)
    assert np.array_equal(_parts(a, 3), a)
    assert _error(_parts(a, 2) @ _parts(b, 2), want) > _allowed(depth)
    # the six products that are taken of three parts: those with h, and m m, come to all of it
    h, m = _parts(a, 1), _parts(a, 2) - _parts(a, 1)
    l, p, q = a - h - m, _parts(b, 1), _parts(b, 2) - _parts(b, 1)  # noqa: E741
    assert _error(h @ b + m @ (p + q) + l @ p, want) < 0.1 * _allowed(depth)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,inner,outer", LINEAR + [(4100, 1030, 4100), (2048, 2048, 2048)])
def test_linear_keeps_its_digits_in_every_tile(cl, rows, inner, outer):
    g = _rng("digits", rows, inner, outer)
    x, w, gy = _normal(g, rows, inner), _normal(g, outer, inner), _normal(g, rows, outer)
    X, W, GY = cl.ClTensor(x), cl.ClTensor(w), cl.ClTensor(gy)
    _check(cl.ClTensor().linear(X, W).float(), x, w.T, "y")
    gx, gw, gx1, gw1 = (cl.ClTensor() for _ in range(4))
    cl.linearBackward(gx, gw, None, GY, X, W)
    cl.linearBackward(gx1, None, None, GY, X, W)
    cl.linearBackward(None, gw1, None, GY, X, W)
    for got in (gx, gx1):
        _check(got.float(), gy, w, "gx")
    for got in (gw, gw1):
        _check(got.float(), gy.T, x, "gw")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,inner,outer,sizes", GROUPED)
def test_groupedmm_keeps_its_digits_in_every_tile(cl, rows, inner, outer, sizes):
    g = _rng("grouped digits", rows, inner, outer)
    x, w, gy = _normal(g, rows, inner), _normal(g, len(sizes), inner, outer), _normal(g, rows, outer)
    X, W, GY = cl.ClTensor(x), cl.ClTensor(w), cl.ClTensor(gy)
    y, gx, gw = cl.ClTensor(rows, outer).fill(0.0), cl.ClTensor(rows, inner).fill(0.0), cl.ClTensor()
    y.groupedmm(X, W, sizes)
    cl.groupedmmBackward(gx, gw, GY, X, W, sizes)
    Y, GX, GW, at = y.float(), gx.float(), gw.float(), 0
    for k, n in enumerate(sizes):
        r = slice(at, at + n)
        at += n
        # a few values say little about a norm
        if n * min(inner, outer) >= 2000:
            _check(Y[r], x[r], w[k], ("y", k))
            _check(GX[r], gy[r], w[k].T, ("gx", k))
        if n and inner * outer >= 2000:
            _check(GW[k], x[r].T, gy[r], ("gw", k))
