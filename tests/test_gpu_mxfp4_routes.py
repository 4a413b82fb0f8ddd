"""MXFP4 layers over groups of rows on every kernel that a plan can choose, with first rows out of order and out of range; large grouped results, which are
stored by kernels of their own; scales from one end to the other; matrices of more than 2^32 bytes and values.

Products of codes are multiples of 2^-2 up to 36. With scales of 2^-1 .. 2^1 they are multiples of 2^-4 up to 144: sums over less than 7281 columns are exact in f32, in any
order, and so is the reference's in f32."""
import numpy as np
import pytest

import iris_c_amd
import mxfp4_reference as mx
from gpu_harness import Dev, ptr_add
from test_gpu_grouped_routes import FIRST

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


def plan_of(groups, rows, k, n):
    return iris_c_amd.load().iris_hip_linear_mxfp4_plan(groups, rows, k, n)


def inputs(rng, rows, k):
    assert k < 7281
    return mx.random_codes(rng, rows, k, 126, 128)


def value(c, s, k):
    return mx.decode(c, s, k).astype(np.float32)


def run(dev, cx, sx, cw, sw, first, groups, rows, k, n, out):
    """y, filled with 7 before, as its bits"""
    y0 = np.full((rows, n), 7.0, np.float32) if out == "f32" else np.full((rows, n), 0x40e0, np.uint16)
    dy = dev.put(y0)
    p = [dev.put(a) for a in (cx, sx, cw, sw)]
    if first is None:
        getattr(dev.lib, f"iris_dev_linear_mxfp4_{out}")(dy, *p, rows, k, n)
    else:
        getattr(dev.lib, f"iris_dev_linear_mxfp4_{out}_grouped")(dy, *p, dev.put(first.astype(np.int32)), groups, rows, k, n)
    dev.check()
    got = dev.get(dy, y0.shape, y0.dtype)
    dev.free_all()
    return got


def same(got, want, out):
    return np.array_equal(got, want) if out == "f32" else np.array_equal(mx.bf16_value(got), mx.bf16_value(mx.bf16_round(want)))


# ----------------------------------------------------------------------------------------------------------------- routes
# groups, rows in all, k, n, and the kernel: -1, -2 a few rows, 0 - 3 the smaller tiles, 4 and 5 those of 256 rows; k both of whole k tiles and not
ROUTES = [(2, 64, 256, 64, -1), (3, 65, 71, 66, -1), (2, 2754, 256, 66, -2), (5, 2695, 85, 66, -2), (3, 3949, 256, 65, 0), (3, 4088, 64, 66, 0),
          (2, 8388, 256, 97, 1), (2, 8405, 73, 97, 1), (3, 8269, 1024, 97, 2), (5, 8463, 907, 101, 2), (3, 8270, 256, 193, 3), (5, 200, 80, 5549, 3),
          (8, 258, 256, 4177, 4), (2, 8294, 296, 393, 4), (8, 269, 256, 6195, 5), (5, 273, 268, 9844, 5),
          (79, 688, 256, 8, -1), (72, 64, 9, 8, -1), (82, 12103, 256, 12, -2), (161, 130, 8, 99, -2), (84, 11162, 256, 22, 0), (168, 189, 9, 115, 0),
          (170, 17137, 256, 40, 1), (102, 14858, 16, 33, 1), (70, 8139, 1024, 128, 2), (117, 9741, 856, 67, 2), (109, 16479, 256, 83, 3), (195, 10233, 9, 65, 3),
          (171, 3295, 256, 192, 4), (107, 1829, 248, 340, 4), (156, 2405, 256, 256, 5), (146, 2621, 248, 243, 5)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("kind", FIRST)
@pytest.mark.parametrize("groups,rows,k,n,route", ROUTES)
def test_every_kernel(dev, groups, rows, k, n, route, kind, out):
    assert plan_of(groups, rows, k, n) == route
    rng = np.random.default_rng(groups + rows)
    first = FIRST[kind](rng, rows, groups)
    cx, sx = inputs(rng, rows, k)
    cw, sw = inputs(rng, groups * n, k)
    got = run(dev, cx, sx, cw, sw, first, groups, rows, k, n, out)
    x, w = value(cx, sx, k), value(cw, sw, k).reshape(groups, n, k)
    at = np.clip(np.maximum.accumulate(np.maximum(first, 0)), 0, rows)
    want = np.full((rows, n), 7.0, np.float32)
    for g in range(groups):
        if at[g + 1] > at[g]:
            want[at[g]:at[g + 1]] = x[at[g]:at[g + 1]] @ w[g].T
    assert same(got, want, out)


# groups of large results: 100 MB and more, rows of 16-byte multiples
@pytest.mark.parametrize("first,behind,k,n,out", [([3, 515, 515, 4100, 4611], 7, 512, 12288, "bf16"), ([1, 2, 300, 2300], 0, 512, 12320, "f32"),
                                                  ([0, 1000, 1000, 1001, 5000], 96, 768, 5376, "f32"), ([90, 3000, 3700, 5200], 2, 2304, 10240, "bf16")])
def test_large_grouped_results_are_whole(dev, first, behind, k, n, out):
    """Every value of the result, from rows of x that repeat 24 different ones"""
    first, groups = np.array(first), len(first) - 1
    rows = int(first[-1]) + behind
    assert rows * n * (2 if out == "bf16" else 4) >= 100 << 20 and plan_of(groups, rows, k, n) >= 4
    rng = np.random.default_rng(rows)
    cx, sx = inputs(rng, 24, k)
    cw, sw = inputs(rng, groups * n, k)
    which = rng.integers(0, 24, rows)
    got = run(dev, cx[which], sx[which], cw, sw, first, groups, rows, k, n, out)
    x, w = value(cx, sx, k), value(cw, sw, k).reshape(groups, n, k)
    for g in range(groups):
        a, b = first[g], first[g + 1]
        assert same(got[a:b], (x @ w[g].T)[which[a:b]], out), g
    outside = np.r_[0:first[0], first[-1]:rows]
    assert (got[outside] == (7.0 if out == "f32" else 0x40e0)).all()


def test_large_results_are_whole(dev):
    for rows, n, k, out in ((4352, 12288, 512, "bf16"), (2300, 12320, 512, "f32")):
        rng = np.random.default_rng(n)
        cx, sx = inputs(rng, 24, k)
        cw, sw = inputs(rng, n, k)
        which = rng.integers(0, 24, rows)
        got = run(dev, cx[which], sx[which], cw, sw, None, 1, rows, k, n, out)
        assert same(got, (value(cx, sx, k) @ value(cw, sw, k).T)[which], out)


# ----------------------------------------------------------------------------------------------------------------- scales
ALL = [(2, 2560, 640, -1), (10, 512, 16384, -2), (100, 2560, 2560, 0), (300, 2560, 2560, 1), (500, 2560, 2560, 2), (1000, 2560, 2560, 3), (500, 512, 16384, 4),
       (3000, 768, 5120, 5), (300, 1100, 1400, 0), (1500, 1100, 1400, 3), (1301, 480, 4007, 4)]


@pytest.mark.parametrize("rows,k,n,route", ALL)
def test_scales_from_one_end_to_the_other_meet(dev, rows, k, n, route):
    """Scales 0 .. 254 of x, and of W what makes their product 2^-1 .. 2^1: sums are as exact as with scales around 2^0"""
    assert plan_of(1, rows, k, n) == route
    rng = np.random.default_rng(k)
    nb = mx.blocks(k)
    cx, _ = inputs(rng, rows, k)
    cw, _ = inputs(rng, n, k)
    at = rng.permutation(np.concatenate([[0, 254, 1, 253], rng.integers(0, 255, nb)]))[:nb]
    sx = np.broadcast_to(at, (rows, nb)).astype(np.uint8)
    sw = np.clip(254 - at + rng.integers(-1, 2, (n, nb)), 0, 254).astype(np.uint8)
    got = run(dev, cx, sx, cw, sw, None, 1, rows, k, n, "f32")
    assert np.array_equal(got, (mx.decode(cx, sx, k) @ mx.decode(cw, sw, k).T).astype(np.float32))


@pytest.mark.parametrize("rows,k,n,route", ALL)
def test_the_largest_and_smallest_products(dev, rows, k, n, route):
    """Two rows' scales are 254 and W's too: 2^254, above all floats. Two rows' are 0: 2^-127 times W's 2^127 is 1. The others are 2^-127 times 2^-64: nothing in f32, and
    next to a block of ordinary products they add nothing."""
    assert plan_of(1, rows, k, n) == route
    rng = np.random.default_rng(n)
    nb = mx.blocks(k)
    cx, cw = np.full((rows, nb * 16), 0x22, np.uint8), np.full((n, nb * 16), 0x22, np.uint8)      # ones
    sx, sw = np.full((rows, nb), 127, np.uint8), np.full((n, nb), 127, np.uint8)
    big, small, tiny = rng.permutation(nb)[:3]
    sw[:, [big, small]], sw[:, tiny] = 254, 63
    sx[:, [big, small, tiny]] = 0
    sx[0, big] = 254
    last = k - 32 * (nb - 1)                                          # columns of the last block; its codes behind them are zeros
    for c in (cx, cw):
        c.reshape(-1, nb, 16)[:, -1, (last + 1) // 2:] = 0
        if last % 2:
            c.reshape(-1, nb, 16)[:, -1, last // 2] &= 15
    got = run(dev, cx, sx, cw, sw, None, 1, rows, k, n, "f32")
    tiny_columns = last if tiny == nb - 1 else 32
    assert (got[1:] == k - tiny_columns).all()
    assert np.isposinf(got[0]).all()


# ----------------------------------------------------------------------------------------------------------------- long matrices
@pytest.mark.parametrize("groups,n,rows,route", [(160, 8192, 300, -2), (160, 8192, 2600, 0), (160, 8192, 18000, 3), (20, 65536, 3000, 4)])
def test_weights_of_more_than_four_gigabytes(dev, groups, n, rows, route):
    """4.7 GB of codes; the first group, one behind 2^32 bytes and the last have rows"""
    k = 7168
    nb = mx.blocks(k)
    assert plan_of(groups, rows, k, n) == route
    far, cut = groups * 19 // 20, rows // 3
    assert far * n * nb * 16 > 1 << 32
    used = {0: (1, cut), far: (cut, cut + 1), groups - 1: (cut + 1, rows - 1)}
    first = np.zeros(groups + 1, np.int32)
    first[0], first[1:far + 1], first[far + 1:groups], first[groups] = 1, cut, cut + 1, rows - 1
    rng = np.random.default_rng(rows)
    cx, sx = inputs(rng, rows, k)
    w = {g: inputs(rng, 4096, k) for g in used}                       # repeated over the n rows
    dw, dws = dev.alloc(groups * n * nb * 16), dev.alloc(groups * n * nb)
    for g, codes_and_scales in w.items():
        for d, a in zip((dw, dws), codes_and_scales):
            for part in range(n // 4096):
                dev.lib.iris_dev_upload(ptr_add(d, (g * (n // 4096) + part) * a.nbytes), a.ctypes.data, a.nbytes)
    dy = dev.put(np.full((rows, n), 7.0, np.float32))
    dev.lib.iris_dev_linear_mxfp4_f32_grouped(dy, dev.put(cx), dev.put(sx), dw, dws, dev.put(first), groups, rows, k, n)
    dev.check()
    got = dev.get(dy, (rows, n), np.float32)
    dev.free_all()
    for g, (a, b) in used.items():
        some = np.unique(np.concatenate([rng.integers(a, b, 20), [a, b - 1]]))
        assert np.array_equal(got[some], np.tile(value(cx[some], sx[some], k) @ value(*w[g], k).T, n // 4096)), g
    assert (got[0] == 7).all() and (got[-1] == 7).all() and (got[1:-1] != 7).any(1).all()


@pytest.mark.parametrize("kind,k", [("mxfp4", 256), ("mxfp4", 64), ("mxfp4", 250), ("groups", 256), ("groups", 65), ("mxfp4 groups", 256)])
def test_results_of_more_than_2_32_values(dev, kind, k):
    rows, n, groups = 530000, 8200, 2
    assert rows * n > 1 << 32
    rng = np.random.default_rng(k)
    which = rng.integers(0, 64, rows)
    first = np.array([5, 200000, rows - 3], np.int32)
    weights = groups if "groups" in kind else 1
    dy = dev.alloc(rows * n * 2)
    some = np.unique(np.concatenate([rng.integers(5, rows - 3, 60), [5, 199999, 200000, 523775, 523776, 523777, rows - 4]]))
    fill = np.full(n, 0x40e0, np.uint16)
    outside = [0, 4, rows - 3, rows - 1] if "groups" in kind else []
    for m in outside:
        dev.lib.iris_dev_upload(ptr_add(dy, m * n * 2), fill.ctypes.data, fill.nbytes)
    if kind == "groups":
        x, w = rng.integers(-8, 9, (64, k)).astype(np.float32), rng.integers(-8, 9, (weights, n, k)).astype(np.float32)
        dev.lib.iris_dev_linear_bf16_grouped(dy, dev.put(mx.bf16_round(x)[which]), dev.put(mx.bf16_round(w)), dev.put(first), groups, rows, k, n)
    else:
        cx, sx = inputs(rng, 64, k)
        cw, sw = inputs(rng, weights * n, k)
        x, w = value(cx, sx, k), value(cw, sw, k).reshape(weights, n, k)
        p = [dev.put(a) for a in (cx[which], sx[which], cw, sw)]
        if weights == 2:
            dev.lib.iris_dev_linear_mxfp4_bf16_grouped(dy, *p, dev.put(first), groups, rows, k, n)
        else:
            dev.lib.iris_dev_linear_mxfp4_bf16(dy, *p, rows, k, n)
    dev.check()
    row = {m: dev.get(ptr_add(dy, int(m) * n * 2).value, (n,), np.uint16) for m in [*some, *outside]}
    dev.free_all()
    for m in some:
        want = x[which[m]] @ w[int(m >= 200000) if weights == 2 else 0].T
        assert same(row[m], want, "bf16"), m
    for m in outside:
        assert (row[m] == 0x40e0).all(), m


def test_conversions_of_more_than_2_32_values(dev):
    rows, cols = 530000, 8200
    nb = mx.blocks(cols)
    assert rows * cols > 1 << 32
    rng = np.random.default_rng(0)
    some = np.unique(np.concatenate([rng.integers(0, rows, 40), [0, 523775, 523776, 523777, rows - 1]]))
    host = mx.bf16_round(rng.standard_normal((len(some), cols)).astype(np.float32))
    d, dc, ds, back = dev.alloc(rows * cols * 2), dev.alloc(rows * nb * 16), dev.alloc(rows * nb), dev.alloc(rows * cols * 2)
    for i, m in enumerate(some):
        dev.lib.iris_dev_upload(ptr_add(d, int(m) * cols * 2), np.ascontiguousarray(host[i]).ctypes.data, cols * 2)
    dev.lib.iris_dev_bf16_to_mxfp4(dc, ds, d, cols, rows, cols)
    dev.lib.iris_dev_mxfp4_to_bf16(back, cols, dc, ds, rows, cols)
    dev.check()
    codes, scales = mx.encode(mx.bf16_value(host))
    want = mx.decode(codes, scales, cols).astype(np.float32)
    for i, m in enumerate(some):
        assert np.array_equal(dev.get(ptr_add(dc, int(m) * nb * 16).value, (nb * 16,), np.uint8), codes[i])
        assert np.array_equal(dev.get(ptr_add(ds, int(m) * nb).value, (nb,), np.uint8), scales[i])
        assert np.array_equal(mx.bf16_value(dev.get(ptr_add(back, int(m) * cols * 2).value, (cols,), np.uint16)), want[i])
    dev.free_all()
