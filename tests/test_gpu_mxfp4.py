"""MXFP4 on the GPU: conversions bit for bit against the 64-bit form, linear layers (one weight matrix, and groups of rows with weights of
their own) against float64 products of the values that codes and scales stand for.

Two kinds of inputs for the layers. With scales of 2^-1 .. 2^1 every product is a multiple of 2^-4 and at most 36 * 4, so up to 7281
columns no sum reaches 2^24 of these multiples: f32 sums are exact in any order, and the f32 result has to be the float64 one bit for bit. Scales over many octaves are held to a bound: a sum of n terms in f32 is off by at
most n 2^-23 sum |terms| (a rounding, or a truncation, of 2^-23 a term), and a bf16 result by half a step, 2^-8 |y|, more.
"""
import numpy as np
import pytest

import mxfp4_reference as mx
from gpu_harness import Dev, ptr_add

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


# ------------------------------------------------------------------------------------------------------------ conversions
def special_rows(rng, rows, cols):
    """Blocks of every size of number, ties, zeros of both signs, denormals, the largest floats"""
    x = (rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-20, 20, (rows, cols)))).astype(np.float32)
    flat = x.reshape(-1)
    n = flat.size
    tie = np.array([4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7, 7.999999, -.25, -5, 0., -0.], np.float32)
    at = rng.integers(0, n, max(1, n // 8))
    flat[at] = tie[rng.integers(0, len(tie), at.size)]
    for start, value in ((0, 1e-45), (64, -3e-39), (128, np.finfo(np.float32).max), (192, 0.0), (256, 2.0 ** -126)):
        flat[start:start + 32] *= np.float32(0)
        if start < n:
            flat[start] = value
    return x


SIZES = [(1, 1, 1), (1, 32, 32), (3, 31, 31), (5, 33, 40), (2, 64, 64), (7, 2565, 2600), (4, 1000, 1001), (1, 4096, 4096), (300, 96, 96), (513, 8, 11)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols,ld", SIZES)
def test_to_mxfp4_is_the_definition_bit_for_bit(dev, kind, rows, cols, ld):
    rng = np.random.default_rng(rows * 7919 + cols)
    x = special_rows(rng, rows, ld)
    if kind == "bf16":
        host = mx.bf16_round(x)
        host[(host & 0x7f80) == 0x7f80] = 0x7f7f               # the largest float rounds to infinity: the largest bf16 instead
        x = mx.bf16_value(host)
    else:
        host = x
    codes, scales = mx.encode(x[:, :cols])
    dx = dev.put(host)
    dc, ds = dev.put(np.full(codes.shape, 0xA5, np.uint8)), dev.put(np.full(scales.size + 8, 0x5A, np.uint8))
    getattr(dev.lib, f"iris_dev_{kind}_to_mxfp4")(dc, ds, dx, ld, rows, cols)
    dev.check()
    got_scales = dev.get(ds, scales.size + 8, np.uint8)
    assert np.array_equal(got_scales[:scales.size], scales.reshape(-1))
    assert (got_scales[scales.size:] == 0x5A).all()
    assert np.array_equal(dev.get(dc, codes.shape, np.uint8), codes)
    dev.free_all()


@pytest.mark.parametrize("kind,offset", [("f32", 4), ("f32", 12), ("bf16", 2), ("bf16", 6)])
def test_to_mxfp4_from_rows_that_start_anywhere(dev, kind, offset):
    rng = np.random.default_rng(offset)
    rows, cols, ld = 9, 203, 211
    x = rng.standard_normal((rows, ld)).astype(np.float32)
    host = x if kind == "f32" else mx.bf16_round(x)
    x = x if kind == "f32" else mx.bf16_value(host)
    codes, scales = mx.encode(x[:, :cols])
    d = dev.alloc(host.nbytes + 16)
    dev.lib.iris_dev_upload(ptr_add(d, offset), host.ctypes.data, host.nbytes)
    dc, ds = dev.alloc(codes.size), dev.alloc(scales.size)
    getattr(dev.lib, f"iris_dev_{kind}_to_mxfp4")(dc, ds, ptr_add(d, offset), ld, rows, cols)
    dev.check()
    assert np.array_equal(dev.get(dc, codes.shape, np.uint8), codes) and np.array_equal(dev.get(ds, scales.shape, np.uint8), scales)
    dev.free_all()


def test_every_bf16_value_and_every_place_in_a_block(dev):
    """All finite bf16 values beside a block maximum of every exponent that they can have, and blocks with infinities and NaN"""
    every = np.arange(1 << 16, dtype=np.uint32).astype(np.uint16)
    x = every.reshape(-1, 32)                                   # neighbours share their exponent, most blocks are full
    rng = np.random.default_rng(3)
    x = np.concatenate([x, rng.permutation(every).reshape(-1, 32)])
    codes, scales = mx.encode(mx.bf16_value(x))
    assert (scales == 255).any() and (scales == 0).any()
    dx, dc, ds = dev.put(x), dev.alloc(codes.size), dev.alloc(scales.size)
    dev.lib.iris_dev_bf16_to_mxfp4(dc, ds, dx, 32, len(x), 32)
    dev.check()
    assert np.array_equal(dev.get(ds, scales.shape, np.uint8), scales) and np.array_equal(dev.get(dc, codes.shape, np.uint8), codes)
    dev.free_all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols,ld", SIZES)
def test_back_from_mxfp4(dev, kind, rows, cols, ld):
    rng = np.random.default_rng(rows + cols)
    codes, scales = mx.random_codes(rng, rows, cols, 0, 252)   # 6 2^125 is the largest that both types hold
    scales[rng.random(scales.shape) < 0.1] = 255
    want = mx.decode(codes, scales, cols).astype(np.float32)
    dc, ds = dev.put(codes), dev.put(scales)
    host = np.full((rows, ld), 1.0, np.float32) if kind == "f32" else np.full((rows, ld), 0x3f80, np.uint16)
    d = dev.put(host)
    getattr(dev.lib, f"iris_dev_mxfp4_to_{kind}")(d, ld, dc, ds, rows, cols)
    dev.check()
    got = dev.get(d, host.shape, host.dtype)
    value = got if kind == "f32" else mx.bf16_value(got)
    assert np.array_equal(value[:, :cols], want, equal_nan=True)
    assert (value[:, cols:] == 1.0).all()
    dev.free_all()


@pytest.mark.parametrize("kind,rows,cols", [("bf16", 4100, 13001), ("f32", 4100, 6501)])
def test_conversions_of_more_than_the_cache_keeps(dev, kind, rows, cols):
    """100 MB and more of values go past the Infinity Cache both ways, in kernels of their own; odd rows that start anywhere"""
    rng = np.random.default_rng(cols)
    host = rng.integers(0, 1 << 16, (rows, cols), dtype=np.uint16)
    host[(host & 0x7f80) == 0x7f80] = 0x3f80
    if kind == "f32":
        host = mx.bf16_value(host)
    size = host.nbytes
    assert size >= 100 << 20
    d, nb = dev.put(host), mx.blocks(cols)
    dc, ds, back = dev.alloc(rows * nb * 16), dev.alloc(rows * nb), dev.alloc(size)
    getattr(dev.lib, f"iris_dev_{kind}_to_mxfp4")(dc, ds, d, cols, rows, cols)
    getattr(dev.lib, f"iris_dev_mxfp4_to_{kind}")(back, cols, dc, ds, rows, cols)
    dev.check()
    got = dev.get(back, host.shape, host.dtype)
    codes, scales = dev.get(dc, (rows, nb * 16), np.uint8), dev.get(ds, (rows, nb), np.uint8)
    dev.free_all()
    some = np.unique(np.concatenate([rng.integers(0, rows, 40), [0, 1, rows - 1]]))
    value = host[some] if kind == "f32" else mx.bf16_value(host[some])
    want_codes, want_scales = mx.encode(value)
    assert np.array_equal(codes[some], want_codes) and np.array_equal(scales[some], want_scales)
    want = mx.decode(want_codes, want_scales, cols).astype(np.float32)
    assert np.array_equal(got[some] if kind == "f32" else mx.bf16_value(got[some]), want)


# ----------------------------------------------------------------------------------------------------------------- layers
def run_layer(dev, codes_x, scales_x, codes_w, scales_w, rows, k, n, out, first=None, fill=7.0):
    """y as float32, and the kernel's name"""
    y0 = np.full((rows, n), fill, np.float32)
    dy = dev.put(y0 if out == "f32" else mx.bf16_round(y0))
    p = [dev.put(a) for a in (codes_x, scales_x, codes_w, scales_w)]
    if first is None:
        getattr(dev.lib, f"iris_dev_linear_mxfp4_{out}")(dy, *p, rows, k, n)
    else:
        getattr(dev.lib, f"iris_dev_linear_mxfp4_{out}_grouped")(dy, *p, dev.put(np.asarray(first, np.int32)), len(first) - 1, rows, k, n)
    dev.check()
    got = dev.get(dy, (rows, n), np.float32 if out == "f32" else np.uint16)
    dev.free_all()
    return got if out == "f32" else mx.bf16_value(got)


def exact_inputs(rng, rows, k):
    """Products are multiples of 2^-4 up to 36 * 4: sums over up to 7000 columns are exact in f32"""
    assert k < 7000
    return mx.random_codes(rng, rows, k, 126, 128)


def check_exact(got, want, out):
    want = want.astype(np.float32)
    assert np.array_equal(got, want if out == "f32" else mx.bf16_value(mx.bf16_round(want)))


LAYERS = [(1, 32, 1), (1, 5, 3), (1, 4096, 512), (1, 4096, 515), (2, 64, 16), (3, 100, 17), (16, 256, 128), (17, 288, 129), (33, 1000, 111), (64, 2560, 384),
          (65, 2560, 257), (128, 512, 256), (129, 544, 260), (200, 768, 520), (256, 1024, 1024), (300, 1280, 448), (513, 256, 777), (640, 2560, 1536), (777, 1000, 1111),
          (1024, 2304, 2048), (2050, 640, 2304),
          (256, 512, 192), (257, 768, 256), (511, 512, 200), (768, 1792, 3000)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n", LAYERS)
def test_layer_is_exact_where_f32_sums_are(dev, rows, k, n, out):
    rng = np.random.default_rng(rows * 31 + k + n)
    cx, sx = exact_inputs(rng, rows, k)
    cw, sw = exact_inputs(rng, n, k)
    got = run_layer(dev, cx, sx, cw, sw, rows, k, n, out)
    check_exact(got, mx.decode(cx, sx, k) @ mx.decode(cw, sw, k).T, out)


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n", [(1, 16384, 256), (5, 96, 40), (70, 4096, 320), (300, 9728, 512), (600, 2048, 1100)])
def test_layer_over_many_octaves_of_scales(dev, rows, k, n, out):
    rng = np.random.default_rng(k)
    cx, sx = mx.random_codes(rng, rows, k, 100, 140)
    cw, sw = mx.random_codes(rng, n, k, 110, 150)
    x, w = mx.decode(cx, sx, k), mx.decode(cw, sw, k)
    want = x @ w.T
    bound = (mx.blocks(k) + 32) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)
    got = run_layer(dev, cx, sx, cw, sw, rows, k, n, out)
    if out == "bf16":
        bound = bound + 2.0 ** -8 * (np.abs(want) + bound)
    assert (np.abs(got - want) <= bound).all()


def test_codes_in_every_place_meet_their_counterpart(dev):
    """One code of a row is not zero: y[m, n] picks W[n, place of row m], for every place of three whole k tiles and a tail"""
    k, n = 840, 130
    rng = np.random.default_rng(8)
    cw, sw = exact_inputs(rng, n, k)
    x = np.zeros((k, k), np.float32)
    x[np.arange(k), np.arange(k)] = 1.0
    cx, sx = mx.encode(x)
    got = run_layer(dev, cx, sx, cw, sw, k, k, n, "f32")
    assert np.array_equal(got, mx.decode(cw, sw, k).T.astype(np.float32))


@pytest.mark.parametrize("rows,k,n", [(4, 512, 64), (300, 1024, 512), (40, 1000, 100), (300, 1100, 1400), (500, 512, 16384)])
def test_nan_blocks_reach_their_rows_and_columns_alone(dev, rows, k, n):
    rng = np.random.default_rng(5)
    cx, sx = exact_inputs(rng, rows, k)
    cw, sw = exact_inputs(rng, n, k)
    sx[rows // 2, -1], sw[n // 3, 0] = 255, 255
    got = run_layer(dev, cx, sx, cw, sw, rows, k, n, "f32")
    want = mx.decode(cx, sx, k) @ mx.decode(cw, sw, k).T
    nan = np.zeros((rows, n), bool)
    nan[rows // 2], nan[:, n // 3] = True, True
    assert np.array_equal(np.isnan(got), nan)
    assert np.array_equal(got[~nan], want.astype(np.float32)[~nan])


# ----------------------------------------------------------------------------------------------------------------- groups
GROUPS = {
    "one": [0, 300], "streams": [0, 64, 700], "empty between": [0, 5, 5, 5, 130, 130, 400], "rows left over": [3, 40, 200], "all empty": [0, 0, 0],
    "tiles that just fit": [0, 128, 256, 512, 768], "single rows": list(range(0, 41)), "seventy": [min(3 * i, 150) for i in range(71)],
    "two hundred": sorted(np.random.default_rng(2).integers(0, 500, 201).tolist()), "last only": [0] * 65 + [90],
}


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("k,n", [(256, 256), (1000, 77), (2048, 512)])
@pytest.mark.parametrize("name", GROUPS)
def test_grouped_layer(dev, name, k, n, out):
    first = GROUPS[name]
    groups, rows = len(first) - 1, first[-1] + 9
    if groups * k * n > 1 << 25:
        k = 256
    rng = np.random.default_rng(k + n + groups)
    cx, sx = exact_inputs(rng, rows, k)
    cw, sw = exact_inputs(rng, groups * n, k)
    got = run_layer(dev, cx, sx, cw, sw, rows, k, n, out, first)
    x, w = mx.decode(cx, sx, k), mx.decode(cw, sw, k).reshape(groups, n, k)
    want = np.full((rows, n), 7.0)
    for g in range(groups):
        want[first[g]:first[g + 1]] = x[first[g]:first[g + 1]] @ w[g].T
    check_exact(got, want, out)


# ----------------------------------------------------------------------------------------------------------------- routes
def plan_of(groups, rows, k, n, out):
    import iris_c_amd
    return iris_c_amd.load().iris_hip_linear_mxfp4_plan(groups, rows, k, n)


# rows of each group (one: no groups), k, n, and the kernel: -1, -2 a few rows, 0 - 3 the smaller tiles, 4 and 5 those of 256 rows
ROUTES = [([2], 2560, 640, -1), ([10], 512, 16384, -2), ([100], 2560, 2560, 0), ([300], 2560, 2560, 1), ([500], 2560, 2560, 2), ([1000], 2560, 2560, 3),
          ([500], 512, 16384, 4), ([3000], 768, 5120, 5), ([1, 3, 0, 2], 1024, 512, -1), ([3] * 40, 512, 768, -2), ([60, 32], 4096, 2560, 0),
          ([150, 142], 4096, 2560, 1), ([400, 92], 4096, 2560, 2), ([200] * 9 + [192], 1024, 1024, 3), ([512, 0, 480], 768, 5120, 4), ([300, 2692], 768, 5120, 5),
          ([300], 1100, 1400, 0), ([700], 1100, 1400, 1), ([1000], 1100, 1400, 2), ([1500], 1100, 1400, 3), ([50] * 9 + [42], 1100, 1000, 0),
          ([100] * 6 + [92, 0, 0, 0], 1100, 1000, 1), ([100] * 9 + [92], 1100, 1000, 2), ([200] * 9 + [192], 1100, 1000, 3)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("sizes,k,n,route", ROUTES)
def test_every_route(dev, sizes, k, n, route, out):
    grouped = len(sizes) > 1
    first = np.concatenate([[3], 3 + np.cumsum(sizes)]) if grouped else np.array([0, sizes[0]])
    rows = int(first[-1]) + (5 if grouped else 0)
    assert plan_of(len(sizes), rows, k, n, out) == route
    rng = np.random.default_rng(rows + k)
    cx, sx = exact_inputs(rng, rows, k)
    cw, sw = exact_inputs(rng, len(sizes) * n, k)
    got = run_layer(dev, cx, sx, cw, sw, rows, k, n, out, first if grouped else None)
    x, w = mx.decode(cx, sx, k), mx.decode(cw, sw, k).reshape(len(sizes), n, k)
    want = np.full((rows, n), 7.0)
    for g in range(len(sizes)):
        want[first[g]:first[g + 1]] = x[first[g]:first[g + 1]] @ w[g].T
    check_exact(got, want, out)


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("n", [4007, 8001, 10820])
@pytest.mark.parametrize("k", [256, 512, 768])
@pytest.mark.parametrize("sizes", [[1300], [700, 0, 601], [1, 1299], [1299, 1]])
def test_wide_tiles_at_any_width(dev, sizes, k, n, out):
    """Rows of results that start anywhere, and one k tile, whose scales are fetched with their neighbours'; the groups reach the last row, where there
    are none"""
    rows, groups = sum(sizes), len(sizes)
    assert plan_of(groups, rows, k, n, out) >= 4
    rng = np.random.default_rng(n + k)
    cx, sx = exact_inputs(rng, rows, k)
    cw, sw = exact_inputs(rng, groups * n, k)
    first = np.concatenate([[0], np.cumsum(sizes)])
    got = run_layer(dev, cx, sx, cw, sw, rows, k, n, out, first if groups > 1 else None)
    x, w = mx.decode(cx, sx, k), mx.decode(cw, sw, k).reshape(groups, n, k)
    check_exact(got, np.concatenate([x[first[g]:first[g + 1]] @ w[g].T for g in range(groups)]), out)


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("k", [257, 290, 480, 897, 1504, 3793])
@pytest.mark.parametrize("sizes", [[1301], [700, 0, 601], [1, 1300]])
def test_wide_tiles_of_rows_of_any_length(dev, sizes, k, out):
    """The last k tile is the last eight blocks of a row, of which some have been multiplied before: a NaN among those stays in its row, and values of
    large and small scales are added once"""
    rows, groups, n = sum(sizes), len(sizes), 4007
    assert plan_of(groups, rows, k, n, out) >= 4
    rng = np.random.default_rng(k)
    cx, sx = exact_inputs(rng, rows, k)
    cw, sw = exact_inputs(rng, groups * n, k)
    first = np.concatenate([[0], np.cumsum(sizes)])
    nb = sx.size // rows
    sx = sx.reshape(rows, nb).copy()
    sx[3, nb - 8] = 255                                            # blocks that the last k tile holds for a second time
    sx[4] += 100
    sx[5] -= 60
    got = run_layer(dev, cx, sx, cw, sw, rows, k, n, out, first if groups > 1 else None)
    sx[3, nb - 8] = 127
    x, w = mx.decode(cx, sx, k), mx.decode(cw, sw, k).reshape(groups, n, k)
    want = np.concatenate([x[first[g]:first[g + 1]] @ w[g].T for g in range(groups)])
    assert np.isnan(got[3]).all()
    keep = np.arange(rows) != 3
    check_exact(got[keep], want[keep], out)


@pytest.mark.parametrize("off", [1, 2, 4])
@pytest.mark.parametrize("k", [256, 288, 1024])
def test_wide_tiles_with_scales_that_start_anywhere(dev, k, off):
    rows, n = 1301, 4007
    rng = np.random.default_rng(off)
    cx, sx = exact_inputs(rng, rows, k)
    cw, sw = exact_inputs(rng, n, k)

    def shifted(a):
        d = dev.alloc(a.nbytes + 16)
        dev.lib.iris_dev_upload(ptr_add(d, off), a.ctypes.data, a.nbytes)
        return ptr_add(d, off)

    y = dev.put(np.full(rows * n, 7.0, np.float32))
    dev.lib.iris_dev_linear_mxfp4_f32(y, dev.put(cx), shifted(sx), dev.put(cw), shifted(sw), rows, k, n)
    dev.check()
    got = dev.get(y, (rows, n), np.float32)
    dev.free_all()
    check_exact(got, mx.decode(cx, sx, k) @ mx.decode(cw, sw, k).T, "f32")


@pytest.mark.parametrize("rows,k,n", [(3, 1024, 64), (70, 1024, 512), (300, 768, 512), (500, 512, 16384)])
@pytest.mark.parametrize("off", [1, 2, 3, 4, 8])
def test_scales_and_results_that_start_anywhere(dev, rows, k, n, off):
    """Scales are bytes, and y needs no more than its own type's alignment"""
    rng = np.random.default_rng(off)
    cx, sx = exact_inputs(rng, rows, k)
    cw, sw = exact_inputs(rng, n, k)

    def shifted(a):
        d = dev.alloc(a.nbytes + 16)
        dev.lib.iris_dev_upload(ptr_add(d, off), a.ctypes.data, a.nbytes)
        return ptr_add(d, off)

    y = dev.put(np.full(rows * n + 16, 7.0, np.float32))
    dev.lib.iris_dev_linear_mxfp4_f32(ptr_add(y, 4 * off), dev.put(cx), shifted(sx), dev.put(cw), shifted(sw), rows, k, n)
    dev.check()
    got = dev.get(y, (rows * n + 16,), np.float32)
    dev.free_all()
    assert (got[:off] == 7).all() and (got[off + rows * n:] == 7).all()
    check_exact(got[off:off + rows * n].reshape(rows, n), mx.decode(cx, sx, k) @ mx.decode(cw, sw, k).T, "f32")


def test_results_too_large_for_the_cache_to_keep(dev):
    """Outputs of 100 MB and more leave past the Infinity Cache, from kernels of their own; rows here and there are compared"""
    for rows, n, out in ((4352, 12288, "bf16"), (2300, 12320, "f32")):
        assert rows * n * (2 if out == "bf16" else 4) >= 100 << 20 and plan_of(1, rows, 512, n, out) >= 4
        rng = np.random.default_rng(rows)
        cx, sx = exact_inputs(rng, rows, 512)
        cw, sw = exact_inputs(rng, n, 512)
        got = run_layer(dev, cx, sx, cw, sw, rows, 512, n, out)
        some = np.unique(np.concatenate([rng.integers(0, rows, 24), [0, 255, 256, rows - 1]]))
        check_exact(got[some], mx.decode(cx[some], sx[some], 512) @ mx.decode(cw, sw, 512).T, out)
        assert (got != 7.0).any(1).all()
