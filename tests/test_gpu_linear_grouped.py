"""Linear layers over groups of rows (bf16) against float64 products. Inputs are whole numbers up to 8 on both sides: products up to 64, sums over
up to 2^18 columns stay below 2^24, so the f32 result is exact in any order of summation and has to equal the float64 one bit for bit."""
import numpy as np
import pytest

import mxfp4_reference as mx
from gpu_harness import Dev, ptr_add

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


def whole(rng, *shape):
    return mx.bf16_round(rng.integers(-8, 9, shape).astype(np.float32))


def reference(x, w, first, rows, n, fill=7.0):
    """The rows of each group times its weights; `first` as any whole numbers: the largest up to each place, limited to the matrix"""
    xf, wf = mx.bf16_value(x).astype(np.float64), mx.bf16_value(w).astype(np.float64)
    at = np.clip(np.maximum.accumulate(np.maximum(np.asarray(first, np.int64), 0)), 0, rows)
    want = np.full((rows, n), fill)
    for g in range(len(at) - 1):
        if at[g + 1] > at[g]:
            want[at[g]:at[g + 1]] = xf[at[g]:at[g + 1]] @ wf[g].T
    return want


def run(dev, x, w, first, rows, k, n, out, offset=0, fill=7.0):
    """offset: elements that x, w and y lie behind a 16-byte boundary"""
    y0 = np.full(rows * n + 8, fill, np.float32)
    y0 = y0 if out == "f32" else mx.bf16_round(y0)
    dy = dev.put(y0)

    def put(a):
        d = dev.alloc(a.nbytes + 32)
        dev.lib.iris_dev_upload(ptr_add(d, 2 * offset), np.ascontiguousarray(a).ctypes.data, a.nbytes)
        return ptr_add(d, 2 * offset)

    yoff = offset * y0.itemsize
    getattr(dev.lib, f"iris_dev_linear_{out}_grouped")(ptr_add(dy, yoff), put(x), put(w), dev.put(np.asarray(first, np.int32)), len(first) - 1, rows, k, n)
    dev.check()
    got = dev.get(dy, y0.shape, y0.dtype)
    got = got if out == "f32" else mx.bf16_value(got)
    dev.free_all()
    at = offset
    assert (got[:at] == fill).all() and (got[at + rows * n:] == fill).all()
    return got[at:at + rows * n].reshape(rows, n)


def check(got, want, out):
    want = want.astype(np.float32)
    assert np.array_equal(got, want if out == "f32" else mx.bf16_value(mx.bf16_round(want)))


FIRST = {
    "one": [0, 300], "streams": [0, 64, 700], "empty between": [0, 5, 5, 5, 130, 130, 400], "rows left over": [3, 40, 200], "all empty": [0, 0, 0],
    "tiles that just fit": [0, 128, 256, 512, 768], "single rows": list(range(0, 41)), "seventy": [min(3 * i, 150) for i in range(71)],
    "two hundred": sorted(np.random.default_rng(2).integers(0, 500, 201).tolist()), "last only": [0] * 65 + [90], "one row": [0, 1],
    "long beside short": [0, 1, 1025, 1030],
}


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("k,n", [(64, 8), (512, 256), (1001, 77), (776, 1111), (2560, 512)])
@pytest.mark.parametrize("name", FIRST)
def test_groups(dev, name, k, n, out):
    first = FIRST[name]
    groups, rows = len(first) - 1, first[-1] + 9
    if groups * k * n > 1 << 25:
        k = 64 if k % 64 == 0 else 97
    rng = np.random.default_rng(k + n + groups)
    x, w = whole(rng, rows, k), whole(rng, groups, n, k)
    check(run(dev, x, w, first, rows, k, n, out), reference(x, w, first, rows, n), out)


@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (2, 7, 3), (130, 9, 129), (128, 64, 128), (129, 65, 5)])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_small_and_unaligned(dev, rows, k, n, offset):
    rng = np.random.default_rng(rows + k)
    first = [0, rows // 2, rows]
    x, w = whole(rng, rows, k), whole(rng, 2, n, k)
    for out in ("f32", "bf16"):
        check(run(dev, x, w, first, rows, k, n, out, offset), reference(x, w, first, rows, n), out)


@pytest.mark.parametrize("first", [[0, 50, 20, 90], [-5, 10, 400], [0, 1000, 50], [90, 10, 5], [-9, -3, -1], [2 ** 31 - 1, 0, 5], [-2 ** 31, 64, 2 ** 31 - 1, 3]])
def test_first_rows_out_of_order_or_out_of_range_stay_inside_the_matrix(dev, first):
    rows, k, n = 100, 128, 96
    rng = np.random.default_rng(1)
    x, w = whole(rng, rows, k), whole(rng, len(first) - 1, n, k)
    check(run(dev, x, w, first, rows, k, n, "f32"), reference(x, w, first, rows, n), "f32")


def test_infinities_and_nan_stay_in_their_rows(dev):
    rows, k, n, first = 150, 320, 200, [0, 60, 150]
    rng = np.random.default_rng(4)
    x, w = whole(rng, rows, k), whole(rng, 2, n, k)
    w[1] = mx.bf16_round(rng.integers(1, 9, (n, k)).astype(np.float32))
    x[10, 3], x[70, 319] = 0x7fc0, 0x7f80                          # NaN in a row of group 0, infinity in one of group 1
    got = run(dev, x, w, first, rows, k, n, "f32")
    x2 = x.copy()
    x2[10, 3] = x2[70, 319] = 0
    want = reference(x2, w, first, rows, n)
    assert np.isnan(got[10]).all() and np.isposinf(got[70]).all()
    keep = np.ones(rows, bool)
    keep[[10, 70]] = False
    assert np.array_equal(got[keep], want[keep].astype(np.float32))


@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_random_values_are_as_near_as_f32_sums_are(dev, out):
    """A sum of k products in f32 is off by at most k 2^-23 sum |products|; bf16 results by half a step more"""
    rows, k, n, first = 700, 1536, 320, [0, 180, 700]
    rng = np.random.default_rng(6)
    x, w = mx.bf16_round(rng.standard_normal((rows, k)).astype(np.float32)), mx.bf16_round(rng.standard_normal((2, n, k)).astype(np.float32))
    got, want = run(dev, x, w, first, rows, k, n, out), reference(x, w, first, rows, n)
    size = reference(x & 0x7fff, w & 0x7fff, first, rows, n)
    bound = k * 2.0 ** -23 * size
    if out == "bf16":
        bound = bound + 2.0 ** -8 * (np.abs(want) + bound)
    assert (np.abs(got - want) <= bound).all()


def plan_of(groups, rows, k, n, size):
    import ctypes as C

    import iris_c_amd
    plan = (C.c_int * 3)()
    iris_c_amd.load().iris_hip_linear_grouped_plan(groups, rows, k, n, size, plan)
    return tuple(plan)


# rows of each group, k, n, and the kernel that the layer takes (3 tiles of 256 rows, 2 the smaller tiles, 1 a few rows, 0 any size)
ROUTES = [([1, 0, 2, 1], 1024, 512, 1), ([3] * 40, 512, 768, 1), ([16, 16], 2560, 6144, 1), ([130, 200], 2560, 1536, 2), ([60] * 24, 1024, 1024, 2),
          ([90, 38], 4096, 2560, 2), ([600, 2500], 512, 8192, 3), ([1000, 0, 3000], 512, 6144, 3), ([900, 1200], 1000, 1600, 0)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("sizes,k,n,kernel", ROUTES)
def test_every_route(dev, sizes, k, n, kernel, out):
    first = np.concatenate([[2], 2 + np.cumsum(sizes)])
    rows = int(first[-1]) + 5
    assert plan_of(len(sizes), rows, k, n, 4 if out == "f32" else 2)[0] == kernel
    rng = np.random.default_rng(rows)
    x, w = whole(rng, rows, k), whole(rng, len(sizes), n, k)
    check(run(dev, x, w, first, rows, k, n, out), reference(x, w, first, rows, n), out)


def test_ranges_of_k_leave_rows_in_no_group_alone(dev):
    """A product whose ranges of K are added by a second kernel, which has to find the rows that are in a group"""
    sizes, k, n = [40, 0, 70], 16384, 512
    first = np.concatenate([[7], 7 + np.cumsum(sizes)])
    rows = int(first[-1]) + 20
    assert plan_of(len(sizes), rows, k, n, 2)[0] == 2 and plan_of(len(sizes), rows, k, n, 2)[2] > 1
    rng = np.random.default_rng(3)
    x, w = whole(rng, rows, k), whole(rng, len(sizes), n, k)
    for out in ("f32", "bf16"):
        check(run(dev, x, w, first, rows, k, n, out), reference(x, w, first, rows, n), out)


# rows of each group, odd k, n, kernel and its shape
ODD = [([3, 0, 1], 129, 1001, 1, 1), ([3, 4, 1], 4097, 1001, 1, 1), ([5] * 16, 777, 2560, 1, 2), ([600, 0], 1355, 512, 1, 2), ([3500, 0], 1355, 256, 0, 2), ([70, 81], 1601, 2661, 0, 2), ([1000, 1000], 833, 2561, 0, 4)]


@pytest.mark.parametrize("offset", [0, 1, 2])
@pytest.mark.parametrize("sizes,k,n,kernel,shape", ODD)
def test_rows_that_start_in_the_middle_of_four_bytes(dev, sizes, k, n, kernel, shape, offset):
    first = np.concatenate([[0], np.cumsum(sizes)])
    rows = int(first[-1])
    assert plan_of(len(sizes), rows, k, n, 4)[:2] == (kernel, shape)
    rng = np.random.default_rng(k)
    x, w = whole(rng, rows, k), whole(rng, len(sizes), n, k)
    for out in ("f32", "bf16"):
        check(run(dev, x, w, first, rows, k, n, out, offset), reference(x, w, first, rows, n), out)


@pytest.mark.parametrize("offset", [1, 2, 3, 8])
@pytest.mark.parametrize("rows,k,n", [(3, 1024, 96), (40, 2560, 640), (300, 512, 1024)])
def test_rows_of_even_length_from_any_start(dev, rows, k, n, offset):
    rng = np.random.default_rng(k)
    first = [0, rows // 3, rows]
    x, w = whole(rng, rows, k), whole(rng, 2, n, k)
    for out in ("f32", "bf16"):
        check(run(dev, x, w, first, rows, k, n, out, offset), reference(x, w, first, rows, n), out)
