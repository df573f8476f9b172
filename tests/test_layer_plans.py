"""The choice of kernel for the products of the layer operators, without a device: the shapes that the GPU tests run
reach all of the kernels, and each choice is one that can be launched."""
import ctypes as C

import pytest

from layer_shapes import GROUPED, LINEAR

WHOLE, ROWS, DEPTH = 0, 1, 2
TILES = [(256, 256, 1), (128, 128, 2), (64, 128, 3), (32, 128, 4)]  # rows, columns, blocks to a compute unit


def _plan(lib, ragged, m, n, k, groups=0, few=True, cus=256):
    p = (C.c_int * 4)()
    lib.thcl_dbg_product_plan(ragged, m, n, k, groups, int(few), cus, p)
    return tuple(p)  # kind, blocks, sharers, slices


def _products(rows, inner, outer, sizes=None):
    """the products behind a forward call, the input's gradient and the weights' gradient"""
    if sizes is None:
        return [("forward", WHOLE, rows, outer, inner, 0), ("input", WHOLE, rows, inner, outer, 0), ("weight", WHOLE, outer, inner, rows, 0)]
    g = len(sizes)
    return [("forward", ROWS, rows, outer, inner, g), ("input", ROWS, rows, inner, outer, g), ("weight", DEPTH, inner, outer, rows, g)]


def test_the_tested_shapes_reach_every_kernel(hooks_lib):
    seen = set()
    for shape in LINEAR + GROUPED:
        for what, ragged, m, n, k, g in _products(*shape):
            kind, _, sharers, slices = _plan(hooks_lib, ragged, m, n, k, g, few=what != "weight")
            seen.add((what, ragged, kind, sharers > 1 or slices > 1))
    missing = [(what, ragged, kind) for what, ragged in (("forward", WHOLE), ("input", WHOLE), ("weight", WHOLE), ("forward", ROWS), ("input", ROWS), ("weight", DEPTH))
               for kind in range(4) if not {(what, ragged, kind, False), (what, ragged, kind, True)} & seen]
    missing += [(what, "few rows", kind) for what in ("forward", "input") for kind in range(4, 8)
                if not {(what, r, kind, s) for r in (WHOLE, ROWS) for s in (False, True)} & seen]
    # split over k or not, for each kind (ragged products in the largest tiles are always large enough to share some)
    missing += [(ragged, kind, split) for ragged in (WHOLE, ROWS) for kind in range(4) for split in (False, True)
                if (ragged, kind, split) != (ROWS, 0, False) and not {(what, ragged, kind, split) for what in ("forward", "input", "weight")} & seen]
    missing += [("few rows", kind, split) for kind in range(4, 8) for split in (False, True)
                if not {(what, r, kind, split) for what in ("forward", "input") for r in (WHOLE, ROWS)} & seen]
    assert not missing, missing


@pytest.mark.parametrize("cus", [256, 64, 1])
def test_every_choice_can_be_launched(hooks_lib, cus):
    for ragged in (WHOLE, ROWS, DEPTH):
        for m in (1, 15, 64, 65, 1000, 40000, 2 ** 31 - 70000):
            for n in (1, 130, 5000, 2 ** 20, 2 ** 31 - 70000):
                for k in (1, 17, 4100, 2 ** 31 - 70000):
                    for g in (1, 8, 65535):
                        if ragged == WHOLE and g > 1:
                            continue
                        kind, blocks, sharers, slices = _plan(hooks_lib, ragged, m, n, k, g, few=ragged != DEPTH, cus=cus)
                        assert 0 <= kind < 8 and 1 <= slices <= 32 and 1 <= sharers <= 32
                        assert slices == 1 or 4 * slices * m * n <= 1e9  # they lie in the workspace
                        assert slices == 1 or (k + 15) // 16 >= 4 * slices
                        if kind >= 4:
                            assert ragged == ROWS and g >= m / 64 or m <= 64
                        elif ragged != WHOLE:
                            assert 1 <= blocks <= cus * TILES[kind][2] and slices == 1


def _pair(lib, rows, inner, outer, cus=256):
    p = (C.c_int * 3)()
    lib.thcl_dbg_pair_plan(rows, inner, outer, cus, p)
    return tuple(p)


def test_gradients_share_a_launch(hooks_lib):
    """the tested shapes take two launches and each tile of one, with either product split and whole"""
    plans = [_pair(hooks_lib, *shape) for shape in LINEAR if shape[0] > 64]
    assert {kind for kind, _, _ in plans} == {0, 1, 2, 3}, plans
    shared = {(p > 1, q > 1) for kind, p, q in plans if kind}
    assert shared == {(False, False), (False, True), (True, False), (True, True)}, plans
    for cus in (256, 64, 1):
        for rows in (65, 1000, 40000, 2 ** 31 - 70000):
            for inner in (1, 130, 5000, 2 ** 31 - 70000):
                for outer in (1, 500, 2 ** 20, 2 ** 31 - 70000):
                    kind, p, q = _pair(hooks_lib, rows, inner, outer, cus)
                    if not kind:
                        continue
                    bm, bn, _ = TILES[kind]
                    blocks = -(-rows // bm) * -(-inner // bn) * p + -(-outer // bm) * -(-inner // bn) * q
                    assert blocks <= 1e6 and 4 * (p * rows * inner * (p > 1) + q * outer * inner * (q > 1)) <= 1e9
                    assert (p == 1 or -(-outer // 16) >= 4 * p) and (q == 1 or -(-rows // 16) >= 4 * q)


def test_few_rows_only_where_they_fit(hooks_lib):
    for m in (1, 16, 64):
        assert _plan(hooks_lib, WHOLE, m, 4096, 4096, few=False)[0] < 4
        assert _plan(hooks_lib, WHOLE, m, 4096, 4096)[0] == 4 + (m - 1) // 16
    assert _plan(hooks_lib, WHOLE, 65, 4096, 4096)[0] < 4
