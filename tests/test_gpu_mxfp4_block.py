"""The MXFP4 conversions and the layers over groups of rows together, as a double-stream block uses them: text rows and image rows with weights of
their own, activations converted in front of each layer; eager, captured into a graph and replayed, and two of them on one workspace."""
import ctypes as C

import numpy as np
import pytest

import mxfp4_reference as mx
from gpu_harness import Dev, ptr_add
from test_gpu_graph import Graphs

pytestmark = pytest.mark.gpu
_vp = C.c_void_p


@pytest.fixture(scope="module")
def dev():
    return Dev()


class Block:
    """x (bf16) -> MXFP4 -> W1 of the row's stream -> bf16 -> MXFP4 -> W2 of the stream -> f32, added to the residual rows"""

    def __init__(self, dev, seed, first, behind, hid, inter):
        rng = np.random.default_rng(seed)
        self.dev, self.first, self.hid, self.inter = dev, list(first), hid, inter
        self.groups, self.rows = len(first) - 1, first[-1] + behind
        self.x = mx.bf16_round((rng.standard_normal((self.rows, hid)) * 2).astype(np.float32))
        self.res = rng.standard_normal((self.rows, hid)).astype(np.float32)
        w1 = (rng.standard_normal((self.groups * inter, hid)) / np.sqrt(hid)).astype(np.float32)
        w2 = (rng.standard_normal((self.groups * hid, inter)) / np.sqrt(inter)).astype(np.float32)
        nb1, nb2 = mx.blocks(hid), mx.blocks(inter)
        self.d = dict(x=dev.put(self.x), res=dev.put(self.res), first=dev.put(np.asarray(first, np.int32)), w1=dev.put(w1), w2=dev.put(w2))
        for name, rows, nb in (("w1", self.groups * inter, nb1), ("w2", self.groups * hid, nb2), ("x", self.rows, nb1), ("h", self.rows, nb2)):
            self.d[name + "c"], self.d[name + "s"] = dev.alloc(rows * nb * 16), dev.alloc(rows * nb)
        self.d["h"], self.d["o"] = dev.put(np.zeros((self.rows, inter), np.uint16)), dev.put(np.zeros((self.rows, hid), np.float32))
        d, lib = self.d, dev.lib
        lib.iris_dev_f32_to_mxfp4(d["w1c"], d["w1s"], d["w1"], hid, self.groups * inter, hid)
        lib.iris_dev_f32_to_mxfp4(d["w2c"], d["w2s"], d["w2"], inter, self.groups * hid, inter)
        dev.check()
        self.w1, self.w2 = (mx.decode(*mx.encode(w), w.shape[1]).reshape(self.groups, -1, w.shape[1]) for w in (w1, w2))

    def run(self):
        d, lib, rows = self.d, self.dev.lib, self.rows
        lib.iris_dev_bf16_to_mxfp4(d["xc"], d["xs"], d["x"], self.hid, rows, self.hid)
        lib.iris_dev_linear_mxfp4_bf16_grouped(d["h"], d["xc"], d["xs"], d["w1c"], d["w1s"], d["first"], self.groups, rows, self.hid, self.inter)
        lib.iris_dev_bf16_to_mxfp4(d["hc"], d["hs"], d["h"], self.inter, rows, self.inter)
        lib.iris_dev_linear_mxfp4_f32_grouped(d["o"], d["hc"], d["hs"], d["w2c"], d["w2s"], d["first"], self.groups, rows, self.inter, self.hid)
        lib.iris_dev_residual(d["res"], d["o"], None, rows, self.hid)

    def reset(self):
        for name, a in (("res", self.res), ("h", np.zeros((self.rows, self.inter), np.uint16)), ("o", np.zeros((self.rows, self.hid), np.float32))):
            self.dev.lib.iris_dev_upload(self.d[name], a.ctypes.data, a.nbytes)

    def results(self):
        return (self.dev.get(self.d["h"], (self.rows, self.inter), np.uint16), self.dev.get(self.d["o"], (self.rows, self.hid), np.float32),
                self.dev.get(self.d["res"], (self.rows, self.hid), np.float32))

    def per_group(self, a, w):
        out = np.zeros((self.rows, w.shape[1]))
        for g in range(self.groups):
            out[self.first[g]:self.first[g + 1]] = a[self.first[g]:self.first[g + 1]] @ w[g].T
        return out

    def check(self):
        """Each step against 64 bits on what the device gave the step: sums of n blocks in f32 are off by (n + 32) 2^-23 sum |terms| at most"""
        h, o, res = self.results()
        a = mx.decode(*mx.encode(mx.bf16_value(self.x)), self.hid)
        want, size = self.per_group(a, self.w1), self.per_group(np.abs(a), np.abs(self.w1))
        bound = (mx.blocks(self.hid) + 32) * 2.0 ** -23 * size
        assert (np.abs(mx.bf16_value(h) - want) <= bound + 2.0 ** -8 * (np.abs(want) + bound)).all()
        a = mx.decode(*mx.encode(mx.bf16_value(h)), self.inter)
        want, size = self.per_group(a, self.w2), self.per_group(np.abs(a), np.abs(self.w2))
        assert (np.abs(o - want) <= (mx.blocks(self.inter) + 32) * 2.0 ** -23 * size).all()
        assert np.array_equal(res, self.res + o)
        return h, o, res


SIZES = [([0, 64, 320], 0, 512, 1024), ([0, 77, 401], 3, 384, 800), ([0, 2, 5], 1, 1024, 512), ([0, 512, 1536], 0, 1024, 2048), ([0, 0, 30, 30, 31], 2, 256, 128)]


@pytest.mark.parametrize("first,behind,hid,inter", SIZES)
def test_block(dev, first, behind, hid, inter):
    b = Block(dev, hid, first, behind, hid, inter)
    b.run()
    dev.check()
    got = b.check()
    b.reset()
    b.run()
    for x, y in zip(got, b.results()):
        assert np.array_equal(x, y)                                # a call gives the same bits every time
    dev.free_all()


@pytest.mark.parametrize("first,behind,hid,inter", SIZES[:4])
def test_captured_block_with_other_groups_at_each_replay(dev, first, behind, hid, inter):
    """The graph reads the groups' first rows when it runs; eager work of the program stands between the replays"""
    b = Block(dev, hid + 1, first, behind, hid, inter)
    b.run()
    dev.check()
    g = Graphs()
    run = g.capture(_vp(dev.lib.iris_dev_stream()), b.run)
    dev.check()
    for replay in range(4):
        b.first = [0] + [min(v + 9 * replay, b.rows) if replay % 2 else max(v - 5 * replay, 0) for v in first[1:]]
        at = np.asarray(b.first, np.int32)
        dev.lib.iris_dev_upload(b.d["first"], at.ctypes.data, at.nbytes)
        b.reset()
        assert g.rt.hipGraphLaunch(run, _vp(dev.lib.iris_dev_stream())) == 0
        dev.lib.iris_dev_sync()
        dev.check()
        replayed = b.check()
        b.reset()
        b.run()
        dev.check()
        for x, y in zip(replayed, b.results()):
            assert np.array_equal(x, y), replay
    g.rt.hipGraphExecDestroy(run)
    dev.free_all()


def test_captured_bf16_groups_beside_eager_ones_that_use_the_workspace(dev):
    """Eager, this product cuts K into ranges in the workspace of the linear layers; captured it must not, as the graph may run beside others"""
    import iris_c_amd
    plan = (C.c_int * 3)()
    iris_c_amd.load().iris_hip_linear_grouped_plan(2, 110, 16384, 512, 4, plan)
    assert plan[0] == 2 and plan[2] > 1
    rng = np.random.default_rng(0)
    rows, k, n = 110, 16384, 512
    whole = lambda *s: mx.bf16_round(rng.integers(-8, 9, s).astype(np.float32))  # noqa: E731
    x, w, first = whole(rows, k), whole(2, n, k), np.array([0, 40, 110], np.int32)
    want = np.concatenate([mx.bf16_value(x[a:b]).astype(np.float64) @ mx.bf16_value(w[g]).astype(np.float64).T for g, (a, b) in enumerate(((0, 40), (40, 110)))]).astype(np.float32)
    dx, dw, df = dev.put(x), dev.put(w), dev.put(first)
    y1, y2 = dev.alloc(rows * n * 4), dev.alloc(rows * n * 4)
    call = lambda y: dev.lib.iris_dev_linear_f32_grouped(y, dx, dw, df, 2, rows, k, n)  # noqa: E731
    call(y1)
    dev.check()
    g = Graphs()
    other = _vp()
    assert g.rt.hipStreamCreate(C.byref(other)) == 0
    run = g.capture(_vp(dev.lib.iris_dev_stream()), lambda: call(y1))
    for _ in range(4):
        for y in (y1, y2):
            junk = np.full(rows * n, 3.0, np.float32)
            dev.lib.iris_dev_upload(y, junk.ctypes.data, junk.nbytes)
        assert g.rt.hipGraphLaunch(run, other) == 0               # on another stream, beside eager calls that use the workspace
        for _ in range(3):
            call(y2)
        assert g.rt.hipStreamSynchronize(other) == 0
        dev.lib.iris_dev_sync()
        dev.check()
        assert np.array_equal(dev.get(y1, (rows, n), np.float32), want) and np.array_equal(dev.get(y2, (rows, n), np.float32), want)
    g.rt.hipGraphExecDestroy(run)
    g.rt.hipStreamDestroy(other)
    dev.free_all()


def test_layers_of_the_two_kinds_read_the_same_rows(dev):
    """Whole numbers that MXFP4 holds exactly: the bf16 layer and the MXFP4 layer over the same groups give the same numbers"""
    rng = np.random.default_rng(12)
    first, k, n = [0, 33, 200], 512, 300
    rows = first[-1]
    half = np.array([0, 1, 2, 3, 4, 6, 8, 12], np.float32)
    x = rng.choice(half, (rows, k)) * rng.choice([-1, 1], (rows, k)).astype(np.float32)
    w = rng.choice(half, (2 * n, k)) * rng.choice([-1, 1], (2 * n, k)).astype(np.float32)
    x[:, ::32], w[:, ::32] = 12, 8                                  # every block's scale holds all of them
    lib = dev.lib
    dx, dw, df = dev.put(mx.bf16_round(x)), dev.put(mx.bf16_round(w)), dev.put(np.asarray(first, np.int32))
    nb = mx.blocks(k)
    xc, xs, wc, ws = dev.alloc(rows * nb * 16), dev.alloc(rows * nb), dev.alloc(2 * n * nb * 16), dev.alloc(2 * n * nb)
    lib.iris_dev_bf16_to_mxfp4(xc, xs, dx, k, rows, k)
    lib.iris_dev_bf16_to_mxfp4(wc, ws, dw, k, 2 * n, k)
    y1, y2 = dev.alloc(rows * n * 4), dev.alloc(rows * n * 4)
    lib.iris_dev_linear_f32_grouped(y1, dx, dw, df, 2, rows, k, n)
    lib.iris_dev_linear_mxfp4_f32_grouped(y2, xc, xs, wc, ws, df, 2, rows, k, n)
    dev.check()
    assert np.array_equal(dev.get(y1, (rows, n), np.float32), dev.get(y2, (rows, n), np.float32))
    dev.free_all()


def test_captured_layer_beside_eager_ones_that_copy_scales_into_the_workspace(dev):
    """Rows that are no whole k tiles long: eager, the layer copies its scales into the workspace of the linear layers; captured it must not"""
    import iris_c_amd
    rows, n, layers = 1000, 5001, []
    lib = dev.lib
    for k in (900, 1300):
        assert iris_c_amd.load().iris_hip_linear_mxfp4_plan(1, rows, k, n) >= 4
        rng = np.random.default_rng(k)
        cx, sx = mx.random_codes(rng, rows, k, 126, 128)
        cw, sw = mx.random_codes(rng, n, k, 126, 128)
        layers.append((dev.put(cx), dev.put(sx), dev.put(cw), dev.put(sw), k, (mx.decode(cx, sx, k) @ mx.decode(cw, sw, k).T).astype(np.float32)))
    y1, y2 = dev.alloc(rows * n * 4), dev.alloc(rows * n * 4)
    call = lambda y, layer: lib.iris_dev_linear_mxfp4_f32(y, *layer[:4], rows, layer[4], n)  # noqa: E731
    for layer in layers:                                              # one behind the other through one workspace
        call(y1, layer)
        call(y2, layers[0])
        dev.check()
        assert np.array_equal(dev.get(y1, (rows, n), np.float32), layer[5]) and np.array_equal(dev.get(y2, (rows, n), np.float32), layers[0][5])
    g = Graphs()
    other = _vp()
    assert g.rt.hipStreamCreate(C.byref(other)) == 0
    run = g.capture(_vp(lib.iris_dev_stream()), lambda: call(y1, layers[0]))
    for _ in range(4):
        for y in (y1, y2):
            junk = np.full(rows * n, 3.0, np.float32)
            lib.iris_dev_upload(y, junk.ctypes.data, junk.nbytes)
        assert g.rt.hipGraphLaunch(run, other) == 0
        for _ in range(3):
            call(y2, layers[1])
        assert g.rt.hipStreamSynchronize(other) == 0
        lib.iris_dev_sync()
        dev.check()
        assert np.array_equal(dev.get(y1, (rows, n), np.float32), layers[0][5]) and np.array_equal(dev.get(y2, (rows, n), np.float32), layers[1][5])
    g.rt.hipGraphExecDestroy(run)
    g.rt.hipStreamDestroy(other)
    dev.free_all()
