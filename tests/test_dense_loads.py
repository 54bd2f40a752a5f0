"""CPU: the dense GEMM's loads to LDS stay inside its operands, with nothing but the vector offset in a
buffer's range check, and bring all of them whichever offsets count (the kernel's own load rules, run on the
host for the last tile of each shape)."""
from __future__ import annotations

import ctypes

import pytest


def wrong(pkg, M, n, K):
    if not pkg.LIB_PATH.exists():
        pytest.skip("librlu.so not built")
    bad = ctypes.c_ulonglong(999)
    rc = pkg.lib().rlu_selftest_dense_loads(M, n, K, ctypes.byref(bad))
    return rc, bad.value


# rows around the groups of 8 that a load takes and the tiles of 128, 192 and 256; strips by whole blocks of 128
# columns, which fill a tile or half of it; whole and broken groups of 8 steps, whose row scales go together
@pytest.mark.parametrize("M", [1, 7, 8, 9, 65, 127, 128, 129, 160, 193, 255, 256, 257, 384, 768])
@pytest.mark.parametrize("n", [1, 128, 129, 256, 151936])
@pytest.mark.parametrize("K", [128, 896, 1024, 2560])
def test_loads_stay_inside_the_operands(pkg, M, n, K):
    assert wrong(pkg, M, n, K) == (0, 0)


def test_loads_of_long_rows(pkg):
    assert wrong(pkg, 255, 129, 128 * 1001) == (0, 0)


def test_load_check_refuses_bad_sizes(pkg):
    assert wrong(pkg, 0, 1, 128)[0] == -1 and wrong(pkg, 1, 0, 128)[0] == -1
    assert wrong(pkg, 1, 1, 0)[0] == -1 and wrong(pkg, 1, 2 ** 31 - 1, 128)[0] == -1
    assert wrong(pkg, 1, 1, 200)[0] == -2 and wrong(pkg, 1, 1, 2 ** 22 + 128)[0] == -2
    assert pkg.lib().rlu_selftest_dense_loads(1, 1, 128, None) == -1
