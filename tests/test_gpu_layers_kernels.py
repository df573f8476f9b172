"""The products and norms of the layer operators where their kernels change: shapes that take each of the tiles, split
over k or not, operands whose lines lie far apart or share memory, offsets past 32 bits, and the longest launches.
Tolerances as in test_gpu_layers.py: a sum of K products in any order is off by (K + 3) u sum |a||b| at most, u = 2^-24."""
import zlib

import numpy as np
import pytest

from layer_shapes import GROUPED, LINEAR

pytestmark = pytest.mark.gpu
F = np.float32
U = 2.0 ** -24
EPS = 1e-5


def _rng(*key):
    return np.random.RandomState(zlib.crc32(repr(key).encode()) & 0x7FFFFFFF)


def _normal(rng, *shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(F)


def _product(a, b):
    """a b in fp64, and what fp32 sums may be off by"""
    a, b = a.astype(np.float64), b.astype(np.float64)
    return a @ b, (a.shape[1] + 3) * U * (np.abs(a) @ np.abs(b))


def _within(got, want_and_tol, what):
    want, tol = want_and_tol
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(), float(np.abs(got - want).max()))


@pytest.mark.parametrize("rows,inner,outer", LINEAR)
def test_linear_in_every_tile(cl, rows, inner, outer):
    g = _rng("tiles", rows, inner, outer)
    x, w, gy, b = _normal(g, rows, inner), _normal(g, outer, inner), _normal(g, rows, outer), _normal(g, outer)
    X, W, GY = cl.ClTensor(x), cl.ClTensor(w), cl.ClTensor(gy)
    want, tol = _product(x, w.T)
    pre, y = cl.ClTensor(), cl.ClTensor()
    y.linear(X, W, cl.ClTensor(b), residual=GY, activation="relu", preact=pre)
    _within(pre.float(), (want + b, tol + U * np.abs(want + b)), "preact")
    got = y.float()
    relu = np.maximum(want + b, 0)
    _within(got, (relu + gy, tol + U * np.abs(want + b) + U * np.abs(relu + gy)), "y")
    y.linear(X, W, cl.ClTensor(b), residual=GY, activation="relu", preact=pre)
    assert np.array_equal(y.float().view(np.uint32), got.view(np.uint32))  # the order of sums does not change
    gx, gw, gx1, gw1 = (cl.ClTensor() for _ in range(4))
    cl.linearBackward(gx, gw, None, GY, X, W)
    cl.linearBackward(gx1, None, None, GY, X, W)
    cl.linearBackward(None, gw1, None, GY, X, W)
    want = _product(gy, w)
    _within(gx.float(), want, "gx")
    _within(gx1.float(), want, "gx alone")
    want = _product(gy.T, x)
    _within(gw.float(), want, "gw")
    _within(gw1.float(), want, "gw alone")


@pytest.mark.parametrize("rows,inner,outer", [(150, 300, 260), (628, 820, 1224), (70, 600, 70)])
def test_gradients_together_with_infinities_and_tiny_values(cl, rows, inner, outer):
    """what does not split keeps to its rows and columns of either gradient where both come from one launch"""
    g = _rng("pair", rows, inner, outer)
    x, w, gy = _normal(g, rows, inner), _normal(g, outer, inner), _normal(g, rows, outer)
    gy[3, 5], x[7, 11], w[9, 2] = np.inf, np.nan, -np.inf
    gx, gw = cl.ClTensor(), cl.ClTensor()
    cl.linearBackward(gx, gw, None, cl.ClTensor(gy), cl.ClTensor(x), cl.ClTensor(w))
    for got, a, b in ((gx.float(), gy, w), (gw.float(), gy.T, x)):
        with np.errstate(invalid="ignore"):
            want = a.astype(np.float64) @ b
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
        fine = np.isfinite(want)
        tol = _product(np.where(np.isfinite(a), a, 0), np.where(np.isfinite(b), b, 0))[1]
        _within(np.where(fine, got, 0), (np.where(fine, want, 0), tol), "beside infinities")
    x, w, gy = _normal(g, rows, inner), _normal(g, outer, inner), _normal(g, rows, outer)
    gy[2] = np.clip(gy[2], -3, 3) * F(1e-37)
    gy[2][np.abs(gy[2]) < 1.2e-38] = 0
    w[:, 4] = np.clip(w[:, 4], -3, 3) * F(1e36)
    cl.linearBackward(gx, gw, None, cl.ClTensor(gy), cl.ClTensor(x), cl.ClTensor(w))
    # 1e-38 per term: products and sums below the normal range may round to its grid or to zero
    want, tol = _product(gy, w)
    _within(gx.float(), (want, tol + outer * 1.2e-38), "gx")
    want, tol = _product(gy.T, x)
    _within(gw.float(), (want, tol + rows * 1.2e-38), "gw")


@pytest.mark.parametrize("rows,inner,outer,sizes", GROUPED)
def test_groupedmm_in_every_tile(cl, rows, inner, outer, sizes):
    g = _rng("grouped tiles", rows, inner, outer)
    x, w, gy = _normal(g, rows, inner), _normal(g, len(sizes), inner, outer), _normal(g, rows, outer)
    X, W, GY = cl.ClTensor(x), cl.ClTensor(w), cl.ClTensor(gy)
    y, gx, gw = cl.ClTensor(rows, outer).fill(-3.0), cl.ClTensor(rows, inner).fill(-4.0), cl.ClTensor()
    y.groupedmm(X, W, sizes)
    cl.groupedmmBackward(gx, gw, GY, X, W, sizes)
    Y, GX, GW = y.float(), gx.float(), gw.float()
    at = 0
    for k, n in enumerate(sizes):
        r = slice(at, at + n)
        at += n
        _within(Y[r], _product(x[r], w[k]), ("y", k))
        _within(GX[r], _product(gy[r], w[k].T), ("gx", k))
        _within(GW[k], _product(x[r].T, gy[r]), ("gw", k))
    assert (Y[at:] == -3).all() and (GX[at:] == -4).all()
    y.groupedmm(X, W, sizes)
    gw2 = cl.ClTensor()
    cl.groupedmmBackward(None, gw2, GY, X, W, sizes)
    assert np.array_equal(y.float().view(np.uint32), Y.view(np.uint32)) and np.array_equal(gw2.float().view(np.uint32), GW.view(np.uint32))


@pytest.mark.parametrize("rows,inner,outer", [(150, 300, 260), (700, 96, 256), (20, 300, 70)])
def test_what_does_not_split_in_shared_tiles(cl, rows, inner, outer):
    """infinities keep to their rows and columns, values of every size keep their digits, in tiles whose k is split"""
    g = _rng("special tiles", rows, inner, outer)
    x, w = _normal(g, rows, inner), _normal(g, 2, inner, outer)
    sizes = [rows - 7, 7]
    x[1, inner - 1], w[0, 5, 3], x[rows - 1, 0] = np.inf, -np.inf, np.nan
    got = cl.ClTensor(rows, outer).groupedmm(cl.ClTensor(x), cl.ClTensor(w), sizes).float()
    dense = cl.ClTensor().linear(cl.ClTensor(x), cl.ClTensor(w[0]).t()).float()
    with np.errstate(invalid="ignore"):
        wants = [np.concatenate([x[:-7].astype(np.float64) @ w[0], x[-7:].astype(np.float64) @ w[1]]), x.astype(np.float64) @ w[0]]
    for y, want, ww in ((got, wants[0], w), (dense, wants[1], w[:1].repeat(2, 0))):
        assert np.array_equal(np.isnan(y), np.isnan(want)) and np.array_equal(np.isposinf(y), np.isposinf(want)) and np.array_equal(np.isneginf(y), np.isneginf(want))
        xc, wc = np.where(np.isfinite(x), x, 0), np.where(np.isfinite(ww), ww, 0)
        tol = np.concatenate([_product(xc[:-7], wc[0])[1], _product(xc[-7:], wc[1])[1]])
        fine = np.isfinite(want)
        _within(np.where(fine, y, 0), (np.where(fine, want, 0), tol), "beside infinities")
    # the smallest normal numbers against the largest, in one corner of an otherwise ordinary product
    x, w = _normal(g, rows, inner), _normal(g, 2, inner, outer)
    x[2] = np.clip(x[2], -3, 3) * F(1e-37)
    x[2][np.abs(x[2]) < 1.2e-38] = 0
    w[0, :, 4] = np.clip(w[0, :, 4], -3, 3) * F(1e36)
    got = cl.ClTensor(rows, outer).groupedmm(cl.ClTensor(x), cl.ClTensor(w), sizes).float()
    want = [_product(x[:-7], w[0]), _product(x[-7:], w[1])]
    # 1e-38 per term: products and sums below the normal range may round to its grid or to zero
    _within(got, (np.concatenate([p[0] for p in want]), np.concatenate([p[1] for p in want]) + inner * 1.2e-38), "sizes of every kind")


@pytest.mark.parametrize("rows,inner,outer", [(1, 5, 3), (7, 37, 70), (37, 70, 37), (150, 100, 200), (65, 1000, 130)])
def test_operands_whose_lines_share_memory(cl, rows, inner, outer):
    g = _rng("shared lines", rows, inner, outer)
    x, gy = _normal(g, 1, inner), _normal(g, 1, outer)
    X, GY = cl.ClTensor(x).expand(rows, inner), cl.ClTensor(gy).expand(rows, outer)
    W = cl.ClTensor(_normal(g, outer, inner))
    gw, gb = cl.ClTensor(), cl.ClTensor()
    cl.linearBackward(None, gw, gb, GY, X, W)
    xs, gs = np.repeat(x, rows, 0), np.repeat(gy, rows, 0)
    _within(gw.float(), _product(gs.T, xs), "gw")
    sizes = [rows // 2, rows - rows // 2]
    gw3 = cl.ClTensor()
    cl.groupedmmBackward(None, gw3, GY, X, cl.ClTensor(2, inner, outer).fill(1.0), sizes)
    for k, n in enumerate(sizes):
        _within(gw3.float()[k], _product(xs[:n].T, gs[:n]), ("gw", k))
    # windows of a line: neighbouring rows share all but one element
    line = _normal(g, rows + max(inner, outer))
    L = cl.ClTensor(line)
    xs = np.stack([line[i:i + inner] for i in range(rows)])
    gs = np.stack([line[i:i + outer] for i in range(rows)])
    X, GY = L.strided([rows, inner], [1, 1], 1), L.strided([rows, outer], [1, 1], 1)
    cl.linearBackward(None, gw, None, GY, X, W)
    _within(gw.float(), _product(gs.T, xs), "windows")
    _within(cl.ClTensor().linear(X, W).float(), _product(xs, W.float().T), "windows forward")
    # a weight that repeats along its inputs, with an infinity in one row of it
    v = _normal(g, outer, 1)
    v[outer // 2] = np.inf
    x = np.abs(_normal(g, rows, inner)) + F(0.5)
    y = cl.ClTensor().linear(cl.ClTensor(x), cl.ClTensor(v).expand(outer, inner)).float()
    assert np.isposinf(y[:, outer // 2]).all()
    rest = np.arange(outer) != outer // 2
    _within(y[:, rest], _product(x, np.repeat(v, inner, 1)[rest].T), "repeated weight")


def _far(cl, arr, pitch):
    """arr with `pitch` elements from row to row"""
    r, c = arr.shape
    buf = cl.ClTensor((r - 1) * pitch + c + 8).fill(-5.0)
    v = buf.strided([r, c], [pitch, 1], 3)
    v.copy(cl.ClTensor(arr))
    return v


@pytest.mark.parametrize("rows,inner,outer", [(1, 9, 5), (9, 40, 70), (70, 19, 130)])
def test_lines_far_apart(cl, rows, inner, outer):
    """pitches from 2^21 elements on take a kernel of their own"""
    g = _rng("far", rows, inner, outer)
    x, w, gy = _normal(g, rows, inner), _normal(g, outer, inner), _normal(g, rows, outer)
    pitch = 2 ** 21 + 5
    X, GY = _far(cl, x, pitch), _far(cl, gy, pitch)
    y = _far(cl, np.zeros((rows, outer), dtype=F), pitch)
    b = _normal(g, outer)
    pre = cl.ClTensor()
    y.linear(X, cl.ClTensor(w), cl.ClTensor(b), residual=GY, activation="relu", preact=pre)
    want, tol = _product(x, w.T)
    _within(pre.float(), (want + b, tol + U * np.abs(want + b)), "preact")
    _within(y.float(), (np.maximum(want + b, 0) + gy, tol + 2 * U * (np.abs(want + b) + np.abs(gy))), "y")
    gx, gw = cl.ClTensor(), cl.ClTensor()
    cl.linearBackward(gx, gw, None, GY, X, _far(cl, w, pitch))
    _within(gx.float(), _product(gy, w), "gx")
    _within(gw.float(), _product(gy.T, x), "gw")
    w3 = _normal(g, 2, inner, outer)
    sizes = [rows - rows // 3, rows // 3]
    y3, gx3, gw3 = cl.ClTensor(rows, outer).fill(0.0), cl.ClTensor(rows, inner).fill(0.0), cl.ClTensor()
    y3.groupedmm(X, cl.ClTensor(w3), sizes)
    cl.groupedmmBackward(gx3, gw3, GY, X, cl.ClTensor(w3), sizes)
    at = 0
    for k, n in enumerate(sizes):
        r = slice(at, at + n)
        at += n
        _within(y3.float()[r], _product(x[r], w3[k]), ("y", k))
        _within(gx3.float()[r], _product(gy[r], w3[k].T), ("gx", k))
        _within(gw3.float()[k], _product(x[r].T, gy[r]), ("gw", k))
    # and sizes that do not fit are refused there as well
    y3.fill(7.0)
    with pytest.raises(cl.ClError, match="group sizes"):
        y3.groupedmm(X, cl.ClTensor(w3), [rows, 1])
        cl.synchronize()
    assert (y3.float() == 7).all()


def test_offsets_past_32_bits(cl):
    """2100 rows 2^20 + 4 elements apart: 2.2e9 elements, 8.8 GB, the results in columns beside the operands"""
    rows, inner, outer, pitch = 2100, 48, 70, 2 ** 20 + 4
    g = _rng("long")
    x, w, gy = _normal(g, rows, inner), _normal(g, outer, inner), _normal(g, rows, outer)
    buf = cl.ClTensor(rows, pitch)
    X, Y, GY = buf.narrow(2, 5, inner), buf.narrow(2, 1001, outer), buf.narrow(2, 2001, outer)
    GX = buf.narrow(2, pitch - inner + 1, inner)
    X.copy(cl.ClTensor(x))
    GY.copy(cl.ClTensor(gy))
    Y.linear(X, cl.ClTensor(w), residual=GY, activation="relu")
    want, tol = _product(x, w.T)
    _within(Y.float(), (np.maximum(want, 0) + gy, tol + U * (np.abs(want) + np.abs(gy))), "y")
    gw = cl.ClTensor()
    cl.linearBackward(GX, gw, None, GY, X, cl.ClTensor(w))
    _within(GX.float(), _product(gy, w), "gx")
    _within(gw.float(), _product(gy.T, x), "gw")
    w3, sizes = _normal(g, 3, inner, outer), [1500, 0, 600]
    Y.groupedmm(X, cl.ClTensor(w3), sizes)
    gw3 = cl.ClTensor()
    cl.groupedmmBackward(GX, gw3, GY, X, cl.ClTensor(w3), sizes)
    y3, gx3, gw3 = Y.float(), GX.float(), gw3.float()
    for k, r in ((0, slice(0, 1500)), (2, slice(1500, 2100))):
        _within(y3[r], _product(x[r], w3[k]), ("y", k))
        _within(gx3[r], _product(gy[r], w3[k].T), ("gx", k))
        _within(gw3[k], _product(x[r].T, gy[r]), ("gw", k))
    # layer norm, in columns beside its input
    N = buf.narrow(2, 5001, inner)
    mean, rstd = cl.ClTensor(), cl.ClTensor()
    N.layerNorm(X, eps=EPS, mean=mean, rstd=rstd)
    x64 = x.astype(np.float64)
    h = (x64 - x64.mean(1, keepdims=True)) / np.sqrt(x64.var(1, keepdims=True) + EPS)
    _within(N.float(), (h, 8 * U * np.abs(h) + 2 * U), "norm")


def _check_norm_gradient(gx, h, gyw, rstd, what):
    want = rstd * (gyw - gyw.mean(-1, keepdims=True) - h * (gyw * h).mean(-1, keepdims=True))
    # a dozen roundings of terms no larger than these
    size = np.abs(gyw) + np.abs(gyw).mean(-1, keepdims=True) + np.abs(h) * np.abs(gyw * h).mean(-1, keepdims=True)
    _within(gx, (want, 12 * U * rstd * size), what)


@pytest.mark.parametrize("rows,width", [(1100, w) for w in (1, 3, 5, 64, 65, 96, 130, 256, 500, 777, 1000, 1024, 1537, 2048, 3001, 4096, 4099, 6000, 8192, 8195)]
                         + [(2049, 1537), (3001, 2052), (5003, 24), (2500, 4096)]
                         + [(16500, 1024), (3000, 8192), (4100, 4099), (20001, 840), (280001, 60), (11000, 1537)])
def test_layer_norm_of_many_rows(cl, rows, width):
    """more rows than take part in one launch for all gradients, of every width class, within the caches and past them"""
    g = _rng("rows", rows, width)
    x, gy, w, b = _normal(g, rows, width), _normal(g, rows, width), _normal(g, width), _normal(g, width)
    X, GY, W, B = (cl.ClTensor(a) for a in (x, gy, w, b))
    y, mean, rstd, gx, gw, gb = (cl.ClTensor() for _ in range(6))
    y.layerNorm(X, W, B, EPS, mean=mean, rstd=rstd)
    cl.layerNormBackward(gx, gw, gb, GY, X, W, mean, rstd)
    x64, g64 = x.astype(np.float64), gy.astype(np.float64)
    r = 1 / np.sqrt(x64.var(1, keepdims=True) + EPS)
    h = (x64 - x64.mean(1, keepdims=True)) * r
    want = h * w + b
    # x - mean rounds twice, rstd three times, the product and the sum once
    _within(y.float(), (want, U * (7 * np.abs(h * w) + 2 * np.abs(want)) + 1e-37), "y")
    # the gradient takes x less the rounded mean, off by up to U |mean| rstd in h
    eh = 4 * U * np.abs(h) + U * np.abs(x64.mean(1, keepdims=True)) * r
    gyw = g64 * w
    c1, c2 = gyw.mean(1, keepdims=True), (gyw * h).mean(1, keepdims=True)
    size = np.abs(gyw) + np.abs(gyw).mean(1, keepdims=True) + np.abs(h) * np.abs(gyw * h).mean(1, keepdims=True)
    moved = eh * np.abs(c2) + np.abs(h) * (np.abs(gyw) * eh).mean(1, keepdims=True)
    _within(gx.float(), (r * (gyw - c1 - h * c2), r * (12 * U * size + moved) + 1e-37), "gx")
    _within(gw.float(), ((g64 * h).sum(0), (np.abs(g64) * (eh + 2 * U * np.abs(h))).sum(0) + U * np.abs((g64 * h).sum(0)) + 1e-37), "gw")
    _within(gb.float(), (g64.sum(0), U * np.abs(g64.sum(0)) + 1e-15 * np.abs(g64).sum(0) + 1e-37), "gb")
    # each by itself, and in place of either operand
    gx2, gw2, gb2 = cl.ClTensor(), cl.ClTensor(), cl.ClTensor()
    cl.layerNormBackward(gx2, None, None, GY, X, W, mean, rstd)
    cl.layerNormBackward(None, gw2, None, GY, X, W, mean, rstd)
    cl.layerNormBackward(None, None, gb2, GY, X, W, mean, rstd)
    assert np.array_equal(gx2.float(), gx.float()) and np.array_equal(gw2.float(), gw.float()) and np.array_equal(gb2.float(), gb.float())
    gw2, gb2 = cl.ClTensor(), cl.ClTensor()
    cl.layerNormBackward(GY, gw2, gb2, GY, X, W, mean, rstd)
    assert np.array_equal(GY.float(), gx2.float()) and np.array_equal(gw2.float(), gw.float()) and np.array_equal(gb2.float(), gb.float())
    X.layerNorm(X, W, B, EPS)
    assert np.array_equal(X.float(), y.float())


def test_layer_norm_of_very_wide_rows(cl):
    """more columns than one launch sums with a block to each 32 of them"""
    width = 33_600_001
    g = _rng("wide")
    x, gy = _normal(g, 2, width), _normal(g, 2, width)
    X, GY = cl.ClTensor(x), cl.ClTensor(gy)
    y, mean, rstd, gx, gw, gb = (cl.ClTensor() for _ in range(6))
    y.layerNorm(X, eps=EPS, mean=mean, rstd=rstd)
    cl.layerNormBackward(gx, gw, gb, GY, X, None, mean, rstd)
    x64, g64 = x.astype(np.float64), gy.astype(np.float64)
    r = 1 / np.sqrt(x64.var(1, keepdims=True) + EPS)
    h = (x64 - x64.mean(1, keepdims=True)) * r
    _within(y.float(), (h, 8 * U * np.abs(h) + 2 * U), "y")
    # h is a few roundings off
    _within(gw.float(), ((g64 * h).sum(0), 8 * U * (np.abs(g64) * (np.abs(h) + 0.1)).sum(0)), "gw")
    _within(gb.float(), (g64.sum(0), U * np.abs(g64).sum(0)), "gb")
    # and the gradient's own formula, at the ends and in between
    some = np.r_[0:1000, width // 2:width // 2 + 1000, width - 1000:width]
    c1, c2 = g64.mean(1, keepdims=True), (g64 * h).mean(1, keepdims=True)
    want = r * (g64 - c1 - h * c2)[:, some]
    _within(gx.float()[:, some], (want, 12 * U * (np.abs(g64) + 1)[:, some]), "gx")


def test_layer_norm_of_more_wide_rows_than_blocks(cl):
    """2^20 + 24 rows of 8196 values, all alike: 34 GB of results"""
    rows, width = 2 ** 20 + 24, 8196
    g = _rng("many")
    x, gy = _normal(g, 1, width), _normal(g, 1, width)
    X, GY = cl.ClTensor(x).expand(rows, width), cl.ClTensor(gy).expand(rows, width)
    y, mean, rstd, gx = (cl.ClTensor() for _ in range(4))
    y.layerNorm(X, eps=EPS, mean=mean, rstd=rstd)
    first = y.narrow(1, 1, 1).float()
    for row in (2, 2 ** 20, 2 ** 20 + 1, rows):
        assert np.array_equal(y.narrow(1, row, 1).float(), first)
    assert (mean.float() == mean.float()[0]).all() and (rstd.float() == rstd.float()[0]).all()
    x64, g64 = x.astype(np.float64), gy.astype(np.float64)
    r = 1 / np.sqrt(x64.var(1, keepdims=True) + EPS)
    h = (x64 - x64.mean(1, keepdims=True)) * r
    _within(first, (h, 8 * U * np.abs(h) + 2 * U), "y")
    cl.layerNormBackward(y, None, None, GY, X, None, mean, rstd)
    first = y.narrow(1, 1, 1).float()
    for row in (2, 2 ** 20, 2 ** 20 + 1, rows):
        assert np.array_equal(y.narrow(1, row, 1).float(), first)
    _check_norm_gradient(first, h, g64, r, "gx")


def test_gradient_of_more_biases_than_one_launch_folds(cl):
    width = 17_000_003
    gy = _normal(_rng("biases"), 3, width)
    gb = cl.ClTensor()
    cl.linearBackward(None, None, gb, cl.ClTensor(gy), cl.ClTensor(np.ones((3, 1), dtype=F)), cl.ClTensor(width, 1).fill(1.0))
    want = gy.astype(np.float64).sum(0)
    _within(gb.float(), (want, U * np.abs(want) + 1e-40), "gb")
