"""Linear layers over groups of rows on every kernel, tile and form that a plan can choose, with uneven and empty groups, rows in front of and behind them, and
with first rows out of order and out of range. Whole numbers up to 8 on both sides: every f32 sum is exact, and so is the reference's in f32."""
import ctypes as C

import numpy as np
import pytest

import iris_c_amd
import mxfp4_reference as mx
from gpu_harness import Dev, ptr_add

pytestmark = pytest.mark.gpu

VALUES = np.arange(-8, 9).astype(np.float32)
BITS = mx.bf16_round(VALUES)


@pytest.fixture(scope="module")
def dev():
    return Dev()


def plan_of(groups, rows, k, n, size):
    plan = (C.c_int * 3)()
    iris_c_amd.load().iris_hip_linear_grouped_plan(groups, rows, k, n, size, plan)
    return plan[0], plan[1], plan[2] > 1


# groups, rows in all, k, n, and (kernel, tile, ranges of K): kernels 3 tiles of 256 rows, 2 the smaller tiles, 1 a few rows, 0 any size
FEW = [(8, 177, 512, 3136, (2, 0, False)), (3, 1430, 4224, 128, (2, 0, True)), (5, 93, 512, 6912, (2, 1, False)), (4, 4034, 3136, 192, (2, 1, True)),
       (59, 2294, 512, 832, (2, 2, False)), (4, 5299, 3712, 256, (2, 2, True)), (46, 1094, 512, 1024, (2, 3, False)), (5, 236, 7744, 448, (2, 3, True)),
       (3, 5333, 512, 1024, (2, 4, False)), (4, 3467, 3136, 320, (2, 4, True)), (5, 5630, 512, 1408, (2, 5, False)), (8, 5151, 5824, 256, (2, 5, True)),
       (3, 5254, 576, 1408, (2, 6, False)), (3, 2682, 4416, 448, (2, 6, True)), (2, 3510, 1408, 128, (2, 7, False)), (2, 1528, 3840, 128, (2, 7, True)),
       (3, 3855, 576, 2368, (3, 5, False)), (8, 926, 384, 3312, (3, 6, False)), (3, 555, 512, 13312, (3, 7, False)), (5, 486, 512, 12864, (3, 8, False)),
       (2, 1948, 575, 228, (0, 2, False)), (3, 205, 111, 6786, (0, 4, False)), (5, 40, 777, 515, (1, 1, False)), (9, 33, 264, 6014, (1, 2, False)),
       (64, 4096, 2560, 1536, (2, 1, False))]
MANY = [(79, 8412, 371, 61, (0, 2, False)), (76, 17380, 179, 65, (0, 4, False)), (72, 64, 9, 8, (1, 1, False)), (161, 130, 8, 99, (1, 2, False)),
        (87, 5603, 512, 128, (2, 7, False)), (74, 3376, 2368, 128, (2, 0, True)), (79, 4620, 256, 448, (3, 5, False)), (74, 7587, 384, 320, (3, 6, False)),
        (94, 6857, 256, 448, (3, 7, False)), (79, 6648, 128, 704, (3, 8, False))]


def uneven(rng, rows, groups):
    """First rows of groups of which a sixth are empty, with rows in front of and behind them"""
    share = -np.log(1.0 - rng.random(groups)) * (rng.random(groups) >= 1 / 6)
    share[rng.integers(groups)] += 0.5
    front, behind = min(2, rows - 1), min(5, rows // 8)
    return front + np.concatenate([[0], np.round(np.cumsum(share) / share.sum() * (rows - front - behind))]).astype(np.int64)


def out_of_order(rng, rows, groups):
    """Uneven ones, of which some fall back, among them those behind the 64th"""
    first = uneven(rng, rows, groups)
    back = rng.random(groups + 1) < 0.3
    back[61:70] = back[groups // 2] = True
    first[back] = first[back] * rng.random(back.sum()) - 3
    return first


def out_of_range(rng, rows, groups):
    first = uneven(rng, rows, groups)
    first[0] = -2 ** 31
    first[1:][rng.random(groups) < 0.2] = -5
    first[-1] = 2 ** 31 - 1
    if groups > 64:
        first[groups - 3] = rows + 1000
    return first


FIRST = {"uneven": uneven, "out of order": out_of_order, "out of range": out_of_range}


def layer(dev, groups, rows, k, n, first, out):
    rng = np.random.default_rng(rows + k + n)
    x, w = rng.integers(0, 17, (rows, k), dtype=np.uint8), rng.integers(0, 17, (groups, n, k), dtype=np.uint8)
    y0 = np.full((rows, n), 7.0, np.float32) if out == "f32" else np.full((rows, n), 0x40e0, np.uint16)
    dy = dev.put(y0)
    getattr(dev.lib, f"iris_dev_linear_{out}_grouped")(dy, dev.put(BITS[x]), dev.put(BITS[w]), dev.put(first.astype(np.int32)), groups, rows, k, n)
    dev.check()
    got = dev.get(dy, y0.shape, y0.dtype)
    dev.free_all()
    at = np.clip(np.maximum.accumulate(np.maximum(first, 0)), 0, rows)
    want = np.full((rows, n), 7.0, np.float32)
    for g in range(groups):
        if at[g + 1] > at[g]:
            want[at[g]:at[g + 1]] = VALUES[x[at[g]:at[g + 1]]] @ VALUES[w[g]].T
    assert np.array_equal(got, want) if out == "f32" else np.array_equal(mx.bf16_value(got), mx.bf16_value(mx.bf16_round(want)))


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("kind", FIRST)
@pytest.mark.parametrize("groups,rows,k,n,route", FEW + MANY)
def test_every_kernel_and_tile(dev, groups, rows, k, n, route, kind, out):
    assert plan_of(groups, rows, k, n, 4 if out == "f32" else 2) == route
    if (groups, rows) == (64, 4096) and kind != "uneven":
        pytest.skip("250 million weights: once")
    layer(dev, groups, rows, k, n, FIRST[kind](np.random.default_rng(groups + rows), rows, groups), out)


# rows of each group, n: a block of columns a wave, and two
@pytest.mark.parametrize("sizes,n", [([3, 0, 1], 37), ([5] * 16, 2560)])
@pytest.mark.parametrize("k", [1, 2, 63, 64, 65, 127, 128, 129, 191, 192, 256, 511, 512, 640, 1025])
@pytest.mark.parametrize("x_off,w_off", [(1, 0), (0, 1), (1, 1), (3, 2), (0, 0)])
def test_few_rows_of_matrices_that_start_in_the_middle_of_four_bytes(dev, sizes, n, k, x_off, w_off):
    """x and W apart, in front of and behind them values that are not numbers; every number of steps up to several a wave"""
    groups, rows = len(sizes), sum(sizes) + 1
    first = np.concatenate([[0], np.cumsum(sizes)])
    rng = np.random.default_rng(k)
    x, w = rng.integers(0, 17, (rows, k), dtype=np.uint8), rng.integers(0, 17, (groups, n, k), dtype=np.uint8)

    def put(a, off):
        host = np.full(a.size + 32, 0x7fff, np.uint16)
        host[16 + off:16 + off + a.size] = BITS[a].reshape(-1)
        return ptr_add(dev.put(host), 2 * (16 + off))

    dy = dev.put(np.full((rows, n), 7.0, np.float32))
    dev.lib.iris_dev_linear_f32_grouped(dy, put(x, x_off), put(w, w_off), dev.put(first.astype(np.int32)), groups, rows, k, n)
    dev.check()
    got = dev.get(dy, (rows, n), np.float32)
    dev.free_all()
    want = np.full((rows, n), 7.0, np.float32)
    for g in range(groups):
        want[first[g]:first[g + 1]] = VALUES[x[first[g]:first[g + 1]]] @ VALUES[w[g]].T
    assert np.array_equal(got, want)
