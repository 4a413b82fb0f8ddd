"""Layers for which the kernels of a few rows would need a launch of 2^32 threads or more run on others: groups of a few rows with very many columns, of which
only some have rows (the weights of the others are never read, and stay as the allocation has them). Whole numbers: results are exact."""
import numpy as np
import pytest

import mxfp4_reference as mx
from gpu_harness import Dev, ptr_add

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


def test_grouped_layer_of_a_million_columns(dev):
    groups, rows, k, n = 512, 520, 1, 1048600
    used = {0: (2, 5), 200: (5, 6), 511: (6, 515)}                    # group: its rows
    first = np.zeros(groups + 1, np.int32)
    first[0], first[1:201], first[201:512], first[512] = 2, 5, 6, 515
    rng = np.random.default_rng(0)
    x = rng.integers(-8, 9, rows).astype(np.float32)
    w = {g: rng.integers(-8, 9, n).astype(np.float32) for g in used}
    dx, dw, df = dev.put(mx.bf16_round(x)), dev.alloc(groups * n * 2), dev.put(first)
    for g, v in w.items():
        host = mx.bf16_round(v)
        dev.lib.iris_dev_upload(ptr_add(dw, g * n * 2), host.ctypes.data, host.nbytes)
    dy = dev.put(np.full(rows * n, 0x40e0, np.uint16))                # 7.0
    dev.lib.iris_dev_linear_bf16_grouped(dy, dx, dw, df, groups, rows, k, n)
    dev.check()
    got = dev.get(dy, (rows, n), np.uint16)
    dev.free_all()
    want = {}
    for m in range(rows):
        g = next((g for g, (a, b) in used.items() if a <= m < b), None)
        if g is None:
            assert (got[m] == 0x40e0).all(), m
            continue
        if (g, x[m]) not in want:                                     # products up to 64 are exact in bf16; a sum that starts at +0 is never -0
            want[g, x[m]] = mx.bf16_round(x[m] * w[g] + 0.0)
        assert np.array_equal(got[m], want[g, x[m]]), m


def test_grouped_mxfp4_layer_of_two_million_columns(dev):
    groups, rows, k, n = 275, 322, 2, 1971220
    used = {0: (1, 4), 100: (4, 5), 274: (5, 320)}
    first = np.zeros(groups + 1, np.int32)
    first[0], first[1:101], first[101:275], first[275] = 1, 4, 5, 320
    rng = np.random.default_rng(1)
    cx, sx = mx.random_codes(rng, rows, k, 126, 128)
    cw, sw = mx.random_codes(rng, 4096 + groups, k, 126, 128)         # row r of group g is row g + r % 4096 of these
    turns = -(-n // 4096)
    dx, dxs, df = dev.put(cx), dev.put(sx), dev.put(first)
    dw, dws = dev.alloc(groups * n * 16), dev.alloc(groups * n)
    for g in used:
        for d, a in ((dw, cw), (dws, sw)):
            host = np.ascontiguousarray(np.tile(a[g:g + 4096], (turns, 1))[:n])
            dev.lib.iris_dev_upload(ptr_add(d, g * host.nbytes), host.ctypes.data, host.nbytes)
    dy = dev.put(np.full(rows * n, 0x40e0, np.uint16))
    dev.lib.iris_dev_linear_mxfp4_bf16_grouped(dy, dx, dxs, dw, dws, df, groups, rows, k, n)
    dev.check()
    got = dev.get(dy, (rows, n), np.uint16)
    dev.free_all()
    x, w = mx.decode(cx, sx, k), mx.decode(cw, sw, k)
    for m in range(rows):
        g = next((g for g, (a, b) in used.items() if a <= m < b), None)
        if g is None:
            assert (got[m] == 0x40e0).all(), m
        else:
            want = mx.bf16_round((w[g:g + 4096] @ x[m] + 0.0).astype(np.float32))
            assert np.array_equal(got[m], np.tile(want, turns)[:n]), m


@pytest.mark.parametrize("k", [2 ** 31 - 1, 2 ** 31 - 64])
def test_the_longest_rows(dev, k):
    """Rows of up to 2^31 - 1 values (4 GB), zeros but for some, the last ones among them"""
    rng = np.random.default_rng(0)
    at = np.unique(np.concatenate([rng.integers(0, k, 60), [0, 1, 127, 128, k // 2, k - 129, k - 65, k - 2, k - 1]]))
    values = rng.integers(1, 9, (2, at.size)).astype(np.float32)
    zeros = np.zeros(1 << 27, np.uint16)
    d = []
    for v in values:
        p = dev.alloc(k * 2)
        for start in range(0, k, zeros.size):
            dev.lib.iris_dev_upload(ptr_add(p, 2 * start), zeros.ctypes.data, 2 * min(zeros.size, k - start))
        bits = mx.bf16_round(v)
        for i, b in zip(at, bits):
            one = np.array([b], np.uint16)
            dev.lib.iris_dev_upload(ptr_add(p, 2 * int(i)), one.ctypes.data, 2)
        d.append(p)
    dy = dev.put(np.full(2, 7.0, np.float32))
    dev.lib.iris_dev_linear_f32_grouped(dy, d[0], d[1], dev.put(np.array([0, 1], np.int32)), 1, 1, k, 1)
    dev.check()
    got = dev.get(dy, (2,), np.float32)
    dev.free_all()
    assert got.tolist() == [float((values[0] * values[1]).sum()), 7.0]
