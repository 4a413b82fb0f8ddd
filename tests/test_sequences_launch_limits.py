"""Numbers of rows that 32 bits would not hold on the device, a few below 2^31 of them: calls that large have grids that no launch holds, and are reported before
anything runs. No GPU."""
import ctypes as C

import pytest

import iris_c_amd
from test_sequences_refusals import plan

A = C.c_void_p(4096)                        # an address that nothing is read from
INVALID = 1                                 # hipErrorInvalidValue
TOP = 2 ** 31 - 1


@pytest.fixture(scope="module")
def lib():
    return iris_c_amd.load()


@pytest.mark.parametrize("rows,heads", [(TOP, 1), (TOP - 7, 1), (TOP // 2, 2), (TOP // 60, 60), (2 ** 28, 7)])
@pytest.mark.parametrize("n", [1, 3, 10 ** 6])
def test_packed_rows(lib, rows, heads, n):
    """One kv head: a tile of 8 columns to a workgroup of 256 threads"""
    f = lib.iris_hip_sequences_any
    f.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p] + [C.c_int] * 6 + [C.c_float, C.c_int]
    assert f(None, A, heads, A, heads, A, A, 1, A, None, n, rows, rows, heads, 1, 1, 1.0, 1) == INVALID


@pytest.mark.parametrize("rows,heads", [(TOP, 1), (TOP - 127, 1), (TOP - 254, 1), (TOP // 2, 2), (TOP // 60, 60)])
@pytest.mark.parametrize("n", [1, 3, 10 ** 6])
@pytest.mark.parametrize("causal", [0, 1])
def test_packed_rows_on_the_matrix_cores(lib, rows, heads, n, causal):
    """Where a call's columns and the last tile's width do not fit 32 bits together, its threads do not fit a launch either"""
    for own in (0, 1):
        waves, blocks, parts = plan(lib, n, rows, rows, heads, 1, causal, own)
        height = 16 * waves * blocks
        tiles = (rows * heads + min(n, rows) * (height - 1)) // height
        assert parts == 1
        assert rows * heads + height - 1 < 2 ** 31 or tiles * 64 * waves >= 2 ** 32


@pytest.mark.parametrize("rows", [TOP, TOP - 15, TOP - 62, 2 ** 30])
@pytest.mark.parametrize("n", [1, 3, 10 ** 6])
@pytest.mark.parametrize("head_dim", [1, 64, 128])
def test_cache_rows(lib, rows, n, head_dim):
    """At most 64 rows to a workgroup of 256 threads, K and V each"""
    w, r = lib.iris_hip_cache_write, lib.iris_hip_cache_read
    w.argtypes = [C.c_void_p] * 5 + [C.c_int] * 2 + [C.c_void_p, C.c_int] + [C.c_void_p] * 3 + [C.c_int, C.c_void_p] + [C.c_int] * 4
    r.argtypes = [C.c_void_p] * 3 + [C.c_int] + [C.c_void_p] * 4 + [C.c_int] * 2 + [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p] + [C.c_int] * 4
    for scales in (None, A):
        assert w(None, A, A, scales, scales, 4, 4, A, 2, A, A, A, head_dim, A, n, rows, 1, head_dim) == INVALID
        assert r(None, A, A, head_dim, A, A, scales, scales, 4, 4, A, 2, A, A, n, rows, 1, head_dim) == INVALID
