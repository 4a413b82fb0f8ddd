"""A text through the cache as a program takes it: the prompts of a batch in one call, what they leave in the cache, prompts that go on from
there, and token after token. Every step is one layer's attention on a fused projection: linear, norm and rotation, cache, attention. Each
result is held to float64 over all keys that the sequence has had by then, as the cache keeps them."""
import ctypes as C

import numpy as np
import pytest

import sequences_reference as sr
from gpu_harness import Dev, ptr_add
from test_gpu_graph import Graphs
from test_gpu_paged_cache import Cache, filled, rows

pytestmark = pytest.mark.gpu
HEADS, KV, HD, DIM, PAGE, EPS = 8, 2, 128, 256, 16, 1e-6
COLS = (HEADS + 2 * KV) * HD


@pytest.fixture(scope="module")
def dev():
    return Dev()


class Layer:
    def __init__(self, dev, kind, most):
        rng = np.random.default_rng(3)
        self.dev, self.lib, self.rng = dev, dev.lib, rng
        n = len(most)
        per = -(-max(most) // PAGE)
        self.cache = Cache(dev, kind, n * per, PAGE, KV, HD, rng.permutation(n * per).reshape(n, per))
        self.w = dev.put(sr.bf16_round((rng.standard_normal((COLS, DIM)) / 16).astype(np.float32)))
        self.wq, self.wk = (dev.put((1 + 0.1 * rng.standard_normal(HD)).astype(np.float32)) for _ in "qk")
        angle = np.arange(max(most))[:, None] * 10000.0 ** (-np.arange(HD // 2) / (HD // 2))
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.k, self.v = ([np.zeros((0, KV, HD)) for _ in most] for _ in "kv")       # what the cache holds, in float64
        self.lengths = [0] * n

    def project(self, new):
        """The fused rows of new[g] more tokens of every sequence, normalised and rotated at their positions; on the device and here"""
        at = np.concatenate([np.arange(a, a + b) for a, b in zip(self.lengths, new)]).astype(int)
        total = len(at)
        x = self.dev.put(sr.bf16_round(self.rng.standard_normal((total, DIM)).astype(np.float32)))
        y = self.dev.alloc(total * COLS * 2)
        cos, sin = self.dev.put(self.cos[at]), self.dev.put(self.sin[at])
        self.lib.iris_dev_linear_bf16(y, x, self.w, total, DIM, COLS)
        self.lib.iris_dev_head_norm_rope_qk(y, ptr_add(y, 2 * HEADS * HD), COLS, self.wq, self.wk, cos, sin, total, HEADS, KV, HD, EPS, 1)
        self.dev.check()
        return y, self.dev.get(y, (total, COLS), np.uint16)

    def store(self, new, y, host):
        """Into the cache, here and there"""
        self.lengths = [a + b for a, b in zip(self.lengths, new)]
        first = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.dlengths, self.dfirst, total = self.dev.put(np.asarray(self.lengths, np.int32)), self.dev.put(first), int(first[-1])
        c = self.cache
        one = all(b == 1 for b in new)
        getattr(self.lib, "iris_dev_cache_write_" + c.kind)(*c.where(), c.pages, PAGE, c.dtable, c.table.shape[1], self.dlengths, ptr_add(y, 2 * HEADS * HD),
                                                            ptr_add(y, 2 * (HEADS + KV) * HD), COLS, None if one else self.dfirst, len(new), total, KV, HD)
        self.dev.check()
        for name, from_, to in (("k", HEADS * HD, (HEADS + KV) * HD), ("v", (HEADS + KV) * HD, COLS)):
            x = sr.bf16_value(host[:, from_:to]).astype(np.float64).reshape(total, KV, HD)
            if c.kind == "fp8":
                code, scale = sr.quantise(x)
                x = sr.e4m3_value(code) * sr.scale_value(scale)[..., None]
            held = getattr(self, name)
            for g in range(len(new)):
                held[g] = np.concatenate([held[g], x[first[g]:first[g + 1]]])

    def check(self, new, host, got, rounded, k=None, v=None):
        first = np.concatenate([[0], np.cumsum(new)])
        for g, n in enumerate(new):
            q = sr.bf16_value(host[first[g]:first[g + 1], :HEADS * HD]).astype(np.float64).reshape(n, HEADS, HD)
            kg, vg = (k or self.k)[g], (v or self.v)[g]
            o, w, s = sr.softmax_rows(q, kg, vg, HD ** -0.5, [len(kg) - n + i + 1 for i in range(n)])
            sr.check(sr.bf16_value(got[first[g]:first[g + 1]]).astype(np.float64).reshape(o.shape), (o, sr.bound(o, w, s, HD, rounded)), f"sequence {g}")


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_prompts_then_more_of_them_then_tokens(dev, kind):
    layer = Layer(dev, kind, [150, 60, 130, 40])
    lib, c = dev.lib, layer.cache

    # the prompts: attention within the rows themselves, as the projection leaves them
    new = [70, 1, 33, 5]
    y, host = layer.project(new)
    layer.store(new, y, host)
    total = sum(new)
    out = dev.alloc(total * HEADS * HD * 2)
    lib.iris_dev_attention_sequences(out, HEADS * HD, y, COLS, ptr_add(y, 2 * HEADS * HD), ptr_add(y, 2 * (HEADS + KV) * HD), COLS, layer.dfirst, None, 4, total, total,
                                     HEADS, KV, HD, HD ** -0.5, 1)
    dev.check()
    own = [sr.bf16_value(a).astype(np.float64).reshape(-1, KV, HD) for a in np.split(host[:, HEADS * HD:(HEADS + KV) * HD], np.cumsum(new)[:-1])]
    val = [sr.bf16_value(a).astype(np.float64).reshape(-1, KV, HD) for a in np.split(host[:, (HEADS + KV) * HD:], np.cumsum(new)[:-1])]
    layer.check(new, host, dev.get(out, (total, HEADS * HD), np.uint16), True, own, val)

    # more of each prompt but one: all of the sequence read back, its new rows behind what was there
    new = [40, 30, 0, 20]
    y, host = layer.project(new)
    layer.store(new, y, host)
    total, keys = sum(new), sum(layer.lengths)
    first_key = dev.put(np.concatenate([[0], np.cumsum(layer.lengths)]).astype(np.int32))
    k, v, out = dev.alloc(keys * KV * HD * 2), dev.alloc(keys * KV * HD * 2), dev.alloc(total * HEADS * HD * 2)
    getattr(lib, "iris_dev_cache_read_" + kind)(k, v, KV * HD, *c.where(), c.pages, PAGE, c.dtable, c.table.shape[1], layer.dlengths, first_key, 4, keys, KV, HD)
    lib.iris_dev_attention_sequences(out, HEADS * HD, y, COLS, k, v, KV * HD, layer.dfirst, first_key, 4, total, keys, HEADS, KV, HD, HD ** -0.5, 1)
    dev.check()
    layer.check(new, host, dev.get(out, (total, HEADS * HD), np.uint16), True)

    # token by token
    for _ in range(5):
        y, host = layer.project([1] * 4)
        layer.store([1] * 4, y, host)
        out = dev.alloc(4 * HEADS * HD * 2)
        getattr(lib, "iris_dev_attention_paged_" + kind)(out, HEADS * HD, y, COLS, *c.where(), c.pages, PAGE, c.dtable, c.table.shape[1], layer.dlengths, 4, HEADS, KV, HD,
                                                         HD ** -0.5, None)
        dev.check()
        assert dev.dev.last_kernel() == "fa_paged_hd128"
        layer.check([1] * 4, host, dev.get(out, (4, HEADS * HD), np.uint16), False)
    dev.free_all()


def test_two_captured_calls_with_workspaces_of_their_own_side_by_side(dev):
    """Replayed on two streams at once, eager calls between the replays: every result is the one of the call alone"""
    kv, heads, lib, g = 2, 8, dev.lib, Graphs()
    stream = C.c_void_p(lib.iris_dev_stream())
    graphs, wants, outs = [], [], []
    for i, lengths in enumerate(([4000, 10, 700], [2600, 2600])):
        c = filled(dev, "fp8" if i else "bf16", lengths, 16, kv, 128, seed=10 + i)
        q = rows(30 + i, len(lengths), heads * 128)
        wants.append(c.attend(lengths, q, heads, 0.09))
        dl, dq, do, ws = dev.put(np.asarray(lengths, np.int32)), dev.put(q), dev.put(np.zeros_like(q)), dev.alloc(lib.iris_dev_attention_paged_workspace())

        def call(c=c, dl=dl, dq=dq, do=do, ws=ws, n=len(lengths)):
            getattr(lib, "iris_dev_attention_paged_" + c.kind)(do, heads * 128, dq, heads * 128, *c.where(), c.pages, 16, c.dtable, c.table.shape[1], dl, n, heads, kv, 128,
                                                               0.09, ws)
        graphs.append(g.capture(stream, call))
        outs.append((do, q.shape, call))
    dev.check()
    other = C.c_void_p()
    assert g.rt.hipStreamCreate(C.byref(other)) == 0
    for replay in range(8):
        for do, shape, _ in outs:
            junk = np.full(shape, 0x7f00 + replay, np.uint16)
            lib.iris_dev_upload(do, junk.ctypes.data, junk.nbytes)
        assert g.rt.hipGraphLaunch(graphs[0], stream) == 0 and g.rt.hipGraphLaunch(graphs[1], other) == 0
        lib.iris_dev_sync()
        assert g.rt.hipStreamSynchronize(other) == 0
        for (do, shape, _), want in zip(outs, wants):
            assert np.array_equal(dev.get(do, shape, np.uint16), want)
        outs[replay % 2][2]()
        dev.check()
        assert np.array_equal(dev.get(outs[replay % 2][0], outs[replay % 2][1], np.uint16), wants[replay % 2])
    for e in graphs:
        g.rt.hipGraphExecDestroy(e)
    assert g.rt.hipStreamDestroy(other) == 0
    dev.free_all()


@pytest.mark.parametrize("causal", [0, 1])
def test_keys_in_ranges_eager_and_whole_in_a_graph(dev, causal):
    """A few rows over many keys: cut into ranges when eager, whole when captured; both within the bound, and the same bits each time"""
    heads, kv, hd, first, first_key = 8, 2, 128, [0, 5, 9, 30], [0, 4000, 4003, 9000]
    rng = np.random.default_rng(5)
    q, k, v = (sr.bf16_round(rng.standard_normal(s).astype(np.float32)) for s in ((30, heads * hd), (9000, kv * hd), (9000, kv * hd)))
    v[8000, 3] = 0x7f80
    dq, dk, dv, do = dev.put(q), dev.put(k), dev.put(v), dev.put(np.zeros_like(q))
    df, dfk, g, stream = dev.put(np.asarray(first, np.int32)), dev.put(np.asarray(first_key, np.int32)), Graphs(), C.c_void_p(dev.lib.iris_dev_stream())

    def call():
        dev.lib.iris_dev_attention_sequences(do, heads * hd, dq, heads * hd, dk, dv, kv * hd, df, dfk, 3, 30, 9000, heads, kv, hd, hd ** -0.5, causal)
    plan = [C.c_int() for _ in range(3)]
    dev.lib.iris_hip_sequences_plan(3, 30, 9000, heads, kv, causal, 0, *(C.byref(x) for x in plan))
    assert plan[2].value > 1
    call()
    dev.check()
    eager = dev.get(do, q.shape, np.uint16)
    captured = g.capture(stream, call)
    for replay in range(3):
        assert g.rt.hipGraphLaunch(captured, stream) == 0
        dev.lib.iris_dev_sync()
        whole = dev.get(do, q.shape, np.uint16)
        call()
        assert np.array_equal(dev.get(do, q.shape, np.uint16), eager)
        qf, kf, vf = (sr.bf16_value(a).astype(np.float64).reshape(len(a), -1, hd) for a in (q, k, v))
        for got in (eager, whole):
            for (a, b), (c, d) in zip(zip(first, first[1:]), zip(first_key, first_key[1:])):
                have = sr.bf16_value(got[a:b]).astype(np.float64).reshape(b - a, heads, hd)
                if d == 9000:
                    assert (have[:, :heads // kv, 3] == np.inf).all()
                    have[:, :heads // kv, 3] = 0
                clean = np.where(np.isinf(vf[c:d]), 0, vf[c:d])
                o, w, s = sr.softmax_rows(qf[a:b], kf[c:d], clean, hd ** -0.5, [i + 1 + (d - c) - (b - a) if causal else d - c for i in range(b - a)])
                if d == 9000:
                    o[:, :heads // kv, 3] = 0
                sr.check(have, (o, sr.bound(o, w, s, hd, True)))
    g.rt.hipGraphExecDestroy(captured)
    dev.free_all()
