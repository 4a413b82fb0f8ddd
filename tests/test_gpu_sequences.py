"""iris_dev_attention_sequences against float64, sequence by sequence: lengths from none to long ones, grouped heads, causal and not, keys that
begin in front of the rows, rows of any stride and alignment, values that are not numbers where they must not be seen."""
import ctypes as C

import numpy as np
import pytest

import sequences_reference as sr
from gpu_harness import Dev, ptr_add

pytestmark = pytest.mark.gpu
FILL = 0x4123


@pytest.fixture(scope="module")
def dev():
    return Dev()


def make(seed, rows, keys, heads, kv, hd, spread=1.0):
    rng = np.random.default_rng(seed)
    draw = lambda n, h: sr.bf16_round(rng.standard_normal((n, h * hd)).astype(np.float32) * spread)
    return draw(rows, heads), draw(keys, kv), draw(keys, kv)


def run(dev, q, k, v, first, first_key, heads, kv, hd, scale, causal, pad=0, offset=0, kernel=None, fused=False):
    """pad: elements between rows; offset: elements that q, k, v and out lie behind a 16-byte boundary; fused: q | k | v in one buffer"""
    rows, keys = len(q), len(k)

    def put(a, ld):
        b = np.full((max(len(a), 1), ld), 0x7fc0, np.uint16)               # what lies between the rows is not a number
        b[:len(a), :a.shape[1]] = a
        d = dev.alloc(b.nbytes + 64)
        dev.lib.iris_dev_upload(ptr_add(d, 2 * offset), b.ctypes.data, b.nbytes)
        return ptr_add(d, 2 * offset)

    ldo = heads * hd + pad
    out0 = np.full((rows * ldo + 16,), FILL, np.uint16)
    do = dev.put(out0)
    dfirst = dev.put(np.asarray(first, np.int32))
    dkey = dev.put(np.asarray(first_key, np.int32)) if first_key is not None else None
    if fused:
        ldq = ldkv = (heads + 2 * kv) * hd + pad
        dq = put(np.concatenate([q, k, v], 1), ldq)
        dk, dv = ptr_add(dq, 2 * heads * hd), ptr_add(dq, 2 * (heads + kv) * hd)
    else:
        ldq, ldkv = heads * hd + pad, kv * hd + pad
        dq, dk, dv = put(q, ldq), put(k, ldkv), put(v, ldkv)
    dev.lib.iris_dev_attention_sequences(ptr_add(do, 2 * offset), ldo, dq, ldq, dk, dv, ldkv, dfirst, dkey, len(first) - 1, rows, keys,
                                         heads, kv, hd, scale, int(causal))
    dev.check()
    if kernel:
        assert dev.dev.last_kernel() == kernel
    got = dev.get(do, out0.shape, np.uint16)
    dev.free_all()
    assert (got[:offset] == FILL).all() and (got[offset + rows * ldo:] == FILL).all()
    got = got[offset:offset + rows * ldo].reshape(rows, ldo)
    assert (got[:, heads * hd:] == FILL).all(), "what lies between the rows was written"
    return got[:, :heads * hd]


def reference(q, k, v, first, first_key, heads, kv, hd, scale, causal, rounded):
    """(values, how far off they may be) of the rows that are in a sequence; the others NaN"""
    rows, keys = len(q), len(k)
    qf, kf, vf = (sr.bf16_value(a).astype(np.float64).reshape(len(a), -1, hd) for a in (q, k, v))
    out, limit = np.full((rows, heads, hd), np.nan), np.zeros((rows, heads, hd))
    at = sr.spans(first, rows)
    for (a, b), (c, d) in zip(at, sr.spans(first_key, keys) if first_key is not None else at):
        n, m = b - a, d - c
        sees = [i + 1 + m - n if causal else m for i in range(n)]
        o, w, s = sr.softmax_rows(qf[a:b], kf[c:d], vf[c:d], scale, sees)
        out[a:b], limit[a:b] = o, sr.bound(o, w, s, hd, rounded)
    return out.reshape(rows, -1), limit.reshape(rows, -1)


def compare(got, want, what=""):
    out, limit = want
    inside = ~np.isnan(out[:, 0])
    assert (got[~inside] == FILL).all(), "a row outside the sequences was written"
    sr.check(sr.bf16_value(got[inside]).astype(np.float64), (out[inside], limit[inside]), what)


def both(dev, first, first_key, heads, kv, hd, causal, seed=1, rows=None, keys=None, scale=None, spread=1.0, kernel=None, rounded=True, **how):
    rows = first[-1] if rows is None else rows
    keys = (first_key[-1] if first_key is not None else rows) if keys is None else keys
    scale = hd ** -0.5 if scale is None else scale
    q, k, v = make(seed, rows, keys, heads, kv, hd, spread)
    got = run(dev, q, k, v, first, first_key, heads, kv, hd, scale, causal, kernel=kernel, **how)
    compare(got, reference(q, k, v, first, first_key, heads, kv, hd, scale, causal, rounded))


FIRST = {
    "one token": [0, 1], "two": [0, 2], "tile": [0, 64], "a tile and one": [0, 65], "odd": [0, 3, 20, 20, 83, 84, 211], "empty ends": [0, 0, 7, 7],
    "left over": [4, 40, 57], "all empty": [0, 0, 0], "many": list(range(0, 3 * 71, 3)), "long and short": [0, 1, 400, 401, 420],
}


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 2), (6, 2), (5, 1)])
@pytest.mark.parametrize("first", FIRST, ids=str)
def test_sequences(dev, first, heads, kv, causal):
    first = FIRST[first]
    both(dev, first, None, heads, kv, 128, causal, rows=first[-1] + 5, fused=True)


@pytest.mark.parametrize("heads,kv", [(1, 1), (16, 1), (17, 1), (40, 1), (48, 16), (300, 1)])
def test_groups_of_any_size(dev, heads, kv):
    both(dev, [0, 9, 9, 43], None, heads, kv, 128, True)


CONTINUED = {
    "front": ([0, 5, 9], [0, 70, 200]), "one of many": ([0, 1, 2, 3], [0, 63, 64, 193]), "fewer keys than rows": ([0, 40, 50], [0, 17, 80]),
    "no keys": ([0, 5, 9], [0, 0, 130]), "keys left over": ([0, 33], [11, 111]), "long": ([0, 70], [0, 1500]),
}


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv", [(3, 3), (8, 2)])
@pytest.mark.parametrize("case", CONTINUED, ids=str)
def test_keys_that_begin_in_front_of_the_rows(dev, case, heads, kv, causal):
    first, first_key = CONTINUED[case]
    both(dev, first, first_key, heads, kv, 128, causal, rows=first[-1] + 2, keys=first_key[-1] + 9)


@pytest.mark.parametrize("first", [[5, 3, 60], [-4, 20, 10, 50], [0, 10, 900], [70, 80], [2 ** 31 - 1, 0, 5], [-2 ** 31, -7, 30, -1, 40]], ids=str)
@pytest.mark.parametrize("use_keys", [False, True])
def test_first_rows_out_of_order_and_out_of_range(dev, first, use_keys):
    both(dev, first, list(reversed(first)) if use_keys else None, 4, 2, 128, True, rows=64, keys=50 if use_keys else None)


def test_first_rows_out_of_order_beyond_64_sequences(dev):
    first = [0] + [7 + 5 * (i % 13) + i for i in range(150)] + [3, 900]
    both(dev, first, None, 2, 1, 128, True, rows=190)
    both(dev, first, first[::-1], 2, 1, 128, True, rows=190, keys=170)


@pytest.mark.parametrize("hd", [1, 7, 64, 80, 96, 129, 256, 513])
@pytest.mark.parametrize("causal", [False, True])
def test_other_head_sizes(dev, hd, causal):
    both(dev, [0, 3, 40, 41, 110], None, 4, 2, hd, causal, rounded=False, kernel="attention_sequences_generic")


@pytest.mark.parametrize("pad,offset", [(0, 1), (3, 0), (4, 0), (8, 0), (24, 8), (1, 3)])
def test_strides_and_alignments(dev, pad, offset):
    both(dev, [0, 30, 99], None, 4, 2, 128, True, pad=pad, offset=offset)
    both(dev, [0, 30, 99], [0, 60, 170], 4, 2, 128, True, pad=pad, offset=offset)


@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_scales_that_are_not_positive(dev, scale):
    both(dev, [0, 30, 99], None, 4, 2, 128, True, scale=scale, rounded=False, kernel="attention_sequences_generic")


@pytest.mark.parametrize("spread", [1e-3, 6.0])
def test_flat_and_sharp_softmax(dev, spread):
    both(dev, [0, 130, 200], None, 4, 2, 128, True, spread=spread)
    both(dev, [0, 130, 200], None, 4, 2, 128, False, spread=spread)


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("where", ["key", "value", "both"])
def test_what_a_row_does_not_see_has_no_part_in_it(dev, where, bad, hd):
    """Rows of one sequence from `cut` on are not numbers in K or V: the rows in front of them, and the other sequences, are as without."""
    heads, kv, first, rows = 8, 2, [0, 75, 210, 216, 300], 310
    q, k, v = make(5, rows, rows, heads, kv, hd)
    dirty_k, dirty_v = k.copy(), v.copy()
    word = sr.bf16_round(np.float32(bad))
    cuts = [(40, 75), (130, 210), (215, 216), (217, 300), (300, 310)]
    for a, b in cuts:
        if where in ("key", "both"):
            dirty_k[a:b, ::3] = word
        if where in ("value", "both"):
            dirty_v[a:b, 1::5] = word
    args = (first, None, heads, kv, hd, hd ** -0.5, True)
    clean, got = run(dev, q, k, v, *args), run(dev, q, dirty_k, dirty_v, *args)
    untouched = np.ones(rows, bool)
    for a, b in cuts:
        untouched[a:b] = False
    assert np.array_equal(got[untouched], clean[untouched])
    seen = sr.bf16_value(got[~untouched & (np.arange(rows) < 300)]).reshape(-1, heads, hd)
    if where == "value":                # an infinity that is seen comes through as itself, in its dims alone
        dims = np.zeros(kv * hd, bool)
        dims[1::5] = True
        dims = np.repeat(dims.reshape(kv, hd), heads // kv, 0)
        hit, rest = seen[:, dims], seen[:, ~dims]
        assert np.isfinite(rest).all()
        assert np.isnan(hit).all() if np.isnan(bad) else (hit == bad).all()
    elif np.isnan(bad):
        assert np.isnan(seen).all()


def test_infinities_of_both_signs_in_one_sum(dev):
    heads, hd, n = 2, 128, 100
    q, k, v = make(6, n, n, heads, heads, hd)
    v[30, 5], v[60, 5], v[45, 9] = (sr.bf16_round(np.float32(x)) for x in (np.inf, -np.inf, np.nan))
    got = sr.bf16_value(run(dev, q, k, v, [0, n], None, heads, heads, hd, hd ** -0.5, True))
    assert np.isfinite(got[:30]).all() and (got[30:60, 5] == np.inf).all() and np.isnan(got[60:, 5]).all()
    assert np.isfinite(got[:45, 9]).all() and np.isnan(got[45:, 9]).all()
    other = np.ones(heads * hd, bool)
    other[[5, 9]] = False
    assert np.isfinite(got[:, other]).all()


def test_a_row_that_is_not_a_number_is_the_only_one(dev):
    q, k, v = make(7, 90, 90, 4, 2, 128)
    q[33] = 0x7fc0
    args = ([0, 20, 90], None, 4, 2, 128, 128 ** -0.5, True)
    got = sr.bf16_value(run(dev, q, k, v, *args))
    assert np.isnan(got[33]).all() and np.isfinite(np.delete(got, 33, 0)).all()


def test_equal_to_the_plain_entry_on_one_sequence(dev):
    """The result of iris_dev_attention within the two roundings"""
    n, heads, kv, hd = 300, 8, 2, 128
    q, k, v = make(8, n, n, heads, kv, hd)
    got = run(dev, q, k, v, [0, n], None, heads, kv, hd, hd ** -0.5, True)
    ld = (heads + 2 * kv) * hd
    plain, _ = dev.attention(np.concatenate([q, k, v], 1), ld, 0, heads * hd, (heads + kv) * hd, n, n, heads, kv, hd, hd ** -0.5, causal=True)
    _, limit = reference(q, k, v, [0, n], None, heads, kv, hd, hd ** -0.5, True, True)
    assert (np.abs(sr.bf16_value(got).astype(np.float64) - sr.bf16_value(plain)) <= 2 * limit).all()


def test_long_sequences_among_short_ones(dev):
    """Sizes at which rows and keys of several workgroups meet; sampled rows against float64"""
    heads, kv, hd = 8, 2, 128
    lengths = [2500, 1, 700, 64, 1300]
    first = [0] + list(np.cumsum(lengths))
    rows = first[-1]
    q, k, v = make(9, rows, rows, heads, kv, hd)
    rng = np.random.default_rng(0)
    for causal in (True, False):
        got = sr.bf16_value(run(dev, q, k, v, first, None, heads, kv, hd, hd ** -0.5, causal)).astype(np.float64)
        for a, b in zip(first[:-1], first[1:]):
            for i in sorted({0, b - a - 1, *rng.integers(0, b - a, 12)}):
                qf, kf, vf = (sr.bf16_value(x).astype(np.float64).reshape(len(x), -1, hd) for x in (q[a + i:a + i + 1], k[a:b], v[a:b]))
                o, w, s = sr.softmax_rows(qf, kf, vf, hd ** -0.5, [i + 1 if causal else b - a])
                sr.check(got[a + i:a + i + 1].reshape(o.shape), (o, sr.bound(o, w, s, hd, True)), f"row {i} of {b - a}")


def test_the_same_bits_every_time_and_from_a_graph(dev):
    from test_gpu_graph import Graphs
    heads, kv, hd, first = 8, 2, 128, [0, 33, 150, 150, 290]
    q, k, v = make(10, 290, 290, heads, kv, hd)
    want = run(dev, q, k, v, first, None, heads, kv, hd, hd ** -0.5, True)
    dq, dk, dv, do = dev.put(q), dev.put(k), dev.put(v), dev.put(np.zeros_like(q))
    dfirst = dev.put(np.asarray(first, np.int32))
    g, stream = Graphs(), C.c_void_p(dev.lib.iris_dev_stream())

    def call():
        dev.lib.iris_dev_attention_sequences(do, heads * hd, dq, heads * hd, dk, dv, kv * hd, dfirst, None, len(first) - 1, 290, 290,
                                             heads, kv, hd, hd ** -0.5, 1)
    captured = g.capture(stream, call)
    dev.check()
    for replay in range(3):
        junk = np.full_like(q, 0x7f00 + replay)
        dev.lib.iris_dev_upload(do, junk.ctypes.data, junk.nbytes)
        assert g.rt.hipGraphLaunch(captured, stream) == 0
        dev.lib.iris_dev_sync()
        assert np.array_equal(dev.get(do, q.shape, np.uint16), want)
    g.rt.hipGraphExecDestroy(captured)
    dev.free_all()


def parts(dev, n, rows, keys, heads, kv, causal, own=False):
    out = [C.c_int() for _ in range(3)]
    dev.lib.iris_hip_sequences_plan(n, rows, keys, heads, kv, int(causal), int(own), *(C.byref(x) for x in out))
    return out[2].value


def ends(lengths):
    return [int(x) for x in np.concatenate([[0], np.cumsum(lengths)])]


CUT = {
    "one row": ([1], [20011], 4, 1), "uneven": ([5, 0, 130, 1, 33], [4000, 77, 64, 1, 9000], 6, 3), "fewer keys than rows": ([40, 20], [10, 5000], 8, 8),
    "no keys": ([3, 9, 4], [0, 3001, 0], 16, 2), "65 sequences": ([1] * 65, [1 + 97 * (i % 41) for i in range(65)], 2, 1), "150 sequences": ([1] * 150, [0] * 90 + [4400] * 60, 1, 1),
    "several tiles": ([300, 77], [3003, 2100], 5, 1), "ten kv heads": ([17], [2222], 20, 10),
    "more tiles than half the parts": ([10] * 12, [50, 5000, 64, 700, 12, 900, 130, 0, 1500, 800, 10, 600], 24, 24),
}


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", CUT, ids=str)
def test_keys_cut_into_parts(dev, case, causal):
    rows, keys, heads, kv = CUT[case]
    first, first_key = ends(rows), ends(keys)
    assert parts(dev, len(rows), first[-1] + 2, first_key[-1] + 9, heads, kv, causal) > 1
    both(dev, first, first_key, heads, kv, 128, causal, rows=first[-1] + 2, keys=first_key[-1] + 9, kernel="fa_sequences_hd128")


def test_own_keys_cut_into_parts(dev):
    assert parts(dev, 1, 2777, 2777, 1, 1, True, True) > 1
    both(dev, [5, 2770], None, 1, 1, 128, True, rows=2777, fused=True)


def test_infinities_behind_the_limit_where_keys_are_cut(dev):
    """Each in a dim of its own, near the limits of 90 rows, whose columns and tiles end at several places: infinite for the rows that see it"""
    n, m, heads = 90, 2300, 2
    assert parts(dev, 1, n, m, heads, heads, True) > 1
    q, k, v = make(4, n, m, heads, heads, 128)
    clean = v.copy()
    at = [0, 3, 31, 32, 40, 57, 58, 63, 64, 88, 89]
    for d, i in enumerate(at):
        for h in range(heads):
            v[m - n + i, 128 * h + d] = 0xff80 if d % 2 else 0x7f80
            clean[m - n + i, 128 * h + d] = 0
    got = run(dev, q, k, v, [0, n], [0, m], heads, heads, 128, 128 ** -0.5, True, kernel="fa_sequences_hd128")
    want, limit = reference(q, k, clean, [0, n], [0, m], heads, heads, 128, 128 ** -0.5, True, True)
    have = sr.bf16_value(got).astype(np.float64)
    for d, i in enumerate(at):
        for h in range(heads):
            c = 128 * h + d
            assert (have[i:, c] == (-np.inf if d % 2 else np.inf)).all() and np.isfinite(have[:i, c]).all(), (i, h)
            have[i:, c] = want[i:, c] = 0
    sr.check(have, (want, limit))


def test_lists_of_parts_are_read_anew_by_a_call(dev):
    """A call with many parts, one with few sequences that are cut, one with none: what an earlier one left in the workspace is not read"""
    for rows, keys in (([1] * 30, [3000] * 30), ([7], [9000]), ([2] * 64, [900] * 63 + [1])):
        both(dev, ends(rows), ends(keys), 4, 2, 128, True, seed=len(rows))
    both(dev, [0, 0, 0], [0, 3000, 9000], 4, 2, 128, True, rows=3, keys=9000)
