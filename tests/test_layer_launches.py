"""Products of the layer operators of very many rows or columns: a launch's threads are counted in 32 bits along each
dimension of its grid.  The choice of tiles on the CPU, calls of some 1e9 rows on the GPU."""
import ctypes as C

import numpy as np
import pytest

F = np.float32
THREADS = [512, 512, 256, 256]                                   # of a block of each tile
TILES = [(256, 256), (128, 128), (64, 128), (32, 128)]
SIZES = [1, 2, 3, 17, 64, 65, 1000, 2 ** 16, 2 ** 20, 2 ** 28, 2 ** 29, 2 ** 30 - 1, 2 ** 30, 1_100_000_000, 2 ** 31 - 70000]


@pytest.mark.parametrize("cus", [256, 64, 1])
def test_chosen_tiles_fit_a_launch(hooks_lib, cus):
    fits = 0
    for m in SIZES:
        for n in SIZES:
            if -(-m // 256) * -(-n // 256) * 512 >= 2 ** 32:
                continue                                         # more than 5e11 results
            for k in (1, 5, 1000):
                for few in (0, 1):
                    p = (C.c_int * 4)()
                    hooks_lib.thcl_dbg_product_plan(0, m, n, k, 0, few, cus, p)
                    if p[0] < 4:
                        (bm, bn), threads = TILES[p[0]], THREADS[p[0]]
                        assert -(-m // bm) * -(-n // bn) * threads < 2 ** 32, (m, n, k, p[0])
                        fits += 1
    assert fits > 300


def _same(t, value):
    """every element of a tensor of any size"""
    return t.min() == value and t.max() == value


ROWS = 1_100_000_000


@pytest.mark.gpu
def test_linear_of_a_thousand_million_rows(cl):
    """more than 2^32 threads in tiles of 128 x 128"""
    x, w, b = (cl.ClTensor(np.array(v, dtype=F)) for v in ([[1.5]], [[-2.0]], [0.25]))
    y = cl.ClTensor().linear(x.expand(ROWS, 1), w, b)
    assert y.size() == (ROWS, 1) and _same(y, -2.75)
    gw = cl.ClTensor()
    cl.linearBackward(None, gw, None, x.expand(1, ROWS), x, y)
    assert gw.size() == (ROWS, 1) and _same(gw, 2.25)


@pytest.mark.gpu
def test_far_lines_and_a_thousand_million_rows(cl):
    far = cl.ClTensor(2 ** 21 + 10).fill(0.0).strided([2, 1], [2 ** 21 + 5, 1], 1)
    far.copy(cl.ClTensor(np.array([[3.0], [-1.0]], dtype=F)))
    y = cl.ClTensor().linear(cl.ClTensor(np.array([[0.5]], dtype=F)).expand(ROWS, 1), far)
    assert _same(y.narrow(2, 1, 1), 1.5) and _same(y.narrow(2, 2, 1), -0.5)


@pytest.mark.gpu
def test_far_lines_and_more_columns_than_a_grid_is_high(cl):
    outer = 65536 * 128 + 77
    g = np.random.RandomState(5)
    x, w = g.randint(-8, 9, (3, 2)).astype(F), g.randint(-8, 9, (outer, 2)).astype(F)
    X = cl.ClTensor(2 * (2 ** 21 + 5) + 10).fill(0.0).strided([3, 2], [2 ** 21 + 5, 1], 1)
    X.copy(cl.ClTensor(x))
    assert np.array_equal(cl.ClTensor().linear(X, cl.ClTensor(w)).float(), x @ w.T)
