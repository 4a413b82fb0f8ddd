"""A launch has fewer than 2^32 threads. Grouped and MXFP4 layers take a kernel whose grid is one, where there is such a kernel, and
report the call otherwise. Host arithmetic; no GPU."""
import ctypes as C

import pytest

import iris_c_amd


@pytest.fixture(scope="module")
def lib():
    return C.CDLL(iris_c_amd.LIB_PATH)


def workgroups(groups, rows, out, tm, tn):
    """The most there can be, rounded up to as many for each XCD"""
    some = min(groups, rows)
    n = (rows + some * (tm - 1)) // tm * -(-out // tn)
    return -(-n // 8) * 8


def grouped_threads(groups, rows, out, plan):
    kernel, shape, splits = plan
    if kernel == 1:
        return 256 * workgroups(groups, rows, out, 16, 16 * shape)
    if kernel == 0:
        return 256 * workgroups(groups, rows, out, 32 * shape, 32 * shape)
    if kernel == 3:
        return 512 * workgroups(groups, rows, out, 256, 32 * shape)
    return 512 * splits * workgroups(groups, rows, out, 64, 96)         # no tile of the smaller ones is smaller


MXFP4 = {-1: (16, 16, 256), -2: (16, 32, 256), 0: (32, 32, 256), 1: (64, 64, 256), 2: (64, 128, 256), 3: (128, 128, 512), 4: (256, 192, 512), 5: (256, 256, 512)}


def mxfp4_threads(groups, rows, out, plan):
    tm, tn, threads = MXFP4[plan]
    return threads * workgroups(groups, rows, out, tm, tn)


# groups, rows, in, out: calls that a kernel for a few rows or of small tiles would need more threads for
LARGE = [(512, 520, 1, 1048600), (3139, 3459, 1, 241408), (40215, 87052, 1, 12603), (47824, 2149766, 31, 13816), (1, 4194304, 8, 8200), (2, 2097153, 64, 9000),
         (275, 322, 2, 1971220), (98604, 3657794, 3, 7251), (5555, 141517, 5, 58205)]


@pytest.mark.parametrize("groups,rows,k,n", LARGE)
def test_a_layer_takes_a_kernel_whose_grid_can_be_launched(lib, groups, rows, k, n):
    plan = (C.c_int * 3)()
    for size in (2, 4):
        lib.iris_hip_linear_grouped_plan(groups, rows, k, n, size, plan)
        assert grouped_threads(groups, rows, n, tuple(plan)) < 1 << 32, tuple(plan)
    plan = lib.iris_hip_linear_mxfp4_plan(groups, rows, k, n)
    assert mxfp4_threads(groups, rows, n, plan) < 1 << 32, plan


def test_ordinary_layers_are_far_from_it(lib):
    plan = (C.c_int * 3)()
    for groups in (1, 2, 128):
        for rows in (1, 40, 512, 4608, 50176):
            for k in (32, 1000, 4096, 16384):
                for n in (8, 1111, 4096, 36864):
                    lib.iris_hip_linear_grouped_plan(groups, rows, k, n, 4, plan)
                    assert grouped_threads(groups, rows, n, tuple(plan)) < 1 << 31
                    assert mxfp4_threads(groups, rows, n, lib.iris_hip_linear_mxfp4_plan(groups, rows, k, n)) < 1 << 31
