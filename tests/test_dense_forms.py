"""CPU tests of what the host says about the forms of the dense products."""
import ctypes as C
import random

import pytest

from mortar_amd import _lib
from util import dense_form


def _sizes(n):
    r = random.Random(5)
    return [(int(2 ** r.uniform(0, 15)), 8 * int(2 ** r.uniform(0, 11)), 16 * int(2 ** r.uniform(0, 10))) for _ in range(n)]


def test_e4m3_products_take_the_tiles_that_are_compiled_for_them():
    for M, N, K in _sizes(4000) + [(4096, 11264, 2048), (8192, 8192, 8192), (1 << 16, 8192, 128)]:
        assert dense_form(5, M, N, K)[0] in ((0, 0), (256, 192), (256, 128), (128, 128), (64, 64))


def test_ranges_and_workspaces_agree():
    L = _lib.lib()
    for M, N, K in _sizes(2000):
        tile, ranges = dense_form(1, M, N, K)
        assert tile != (0, 0) and L.mortar_dense_workspace_bytes(M, N, K) == (4 * ranges * M * N if ranges > 1 else 0)
        few, one = dense_form(0, M, N, K)
        assert (few, one) == ((tile, ranges) if few != (0, 0) else ((0, 0), 1)) and (M <= 8 or few != (0, 0))
        tile, ranges = dense_form(5, M, N, K)
        assert L.mortar_fp8_workspace_bytes(M, N, K) == (4 * ranges * M * N if ranges > 1 else 0)
        assert all(dense_form(kind, M, N, K)[1] == 1 for kind in (2, 3, 4))


@pytest.mark.parametrize("bad", [(-1, 8, 8, 8), (6, 8, 8, 8), (0, 0, 8, 8), (0, 8, 0, 8), (0, 8, 8, 0)])
def test_refusals(bad):
    out = [C.byref(C.c_int32()) for _ in range(3)]
    assert _lib.lib().mortar_dense_form_host(*bad, *out) == -1
    assert _lib.lib().mortar_dense_form_host(0, 8, 8, 8, None, *out[1:]) == -1
