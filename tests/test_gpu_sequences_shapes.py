"""Packed attention in every workgroup shape that calls take, each asked of the plan: sampled rows of ragged sequences against float64, and what is not a
number where rows must not see it."""
import ctypes as C

import numpy as np
import pytest

import sequences_reference as sr
from gpu_harness import Dev
from test_gpu_sequences import ends, make, run

pytestmark = pytest.mark.gpu
HD = 128


@pytest.fixture(scope="module")
def dev():
    return Dev()


def plan(dev, n, rows, keys, heads, kv, causal, own):
    out = [C.c_int() for _ in range(3)]
    dev.lib.iris_hip_sequences_plan(n, rows, keys, heads, kv, int(causal), int(own), *(C.byref(x) for x in out))
    return tuple(x.value for x in out)


SHAPES = {
    # shape (waves, blocks, parts), rows, keys (None: the rows'), query heads, kv heads, causal
    "4 x 2 causal": ((4, 2, 1), [2500, 1, 700, 0, 64, 1300], None, 32, 8, True),
    "4 x 2 causal, five to a kv head": ((4, 2, 1), [1900, 33, 0, 1117, 2], None, 30, 6, True),
    "4 x 2 causal, heads of their own": ((4, 2, 1), [1, 1500, 255, 700], None, 24, 24, True),
    "4 x 2 causal, keys in front": ((4, 2, 1), [900, 333, 1, 800], [1500, 340, 900, 800], 32, 8, True),
    "4 x 2 causal, fewer keys than rows": ((4, 2, 1), [900, 333, 1, 800], [500, 340, 0, 800], 32, 8, True),
    "8 x 1": ((8, 1, 1), [301, 0, 77, 622], None, 32, 8, False),
    "8 x 1, heads of their own": ((8, 1, 1), [199] * 9 + [1, 0], None, 24, 24, False),
    "8 x 1, five to a kv head": ((8, 1, 1), [500, 3, 410], None, 30, 6, False),
    "8 x 1, keys of their own": ((8, 1, 1), [300, 77, 622], [400, 1, 777], 32, 8, False),
    "8 x 2": ((8, 2, 1), [1300, 1, 999], None, 32, 8, False),
    "4 x 1 causal": ((4, 1, 1), [400, 30, 0, 201], None, 32, 8, True),
    "4 x 1": ((4, 1, 1), [200, 30, 0, 101], None, 32, 8, False),
    "2 x 1 causal": ((2, 1, 1), [31], None, 32, 8, True),
    "2 x 1": ((2, 1, 1), [17, 14], None, 32, 8, False),
    "cut, causal": ((4, 1, 512), [64, 1, 200, 17], [2064, 900, 4113, 1217], 32, 8, True),
    "cut": ((4, 1, 512), [64, 1, 200, 17], [2064, 900, 4113, 1217], 32, 8, False),
}


@pytest.mark.parametrize("case", SHAPES, ids=str)
def test_shape(dev, case):
    shape, rows, keys, heads, kv, causal = SHAPES[case]
    first, own = ends(rows), keys is None
    first_key = first if own else ends(keys)
    n, m, scale = first[-1], first_key[-1], HD ** -0.5
    assert plan(dev, len(rows), n, m, heads, kv, causal, own) == shape
    q, k, v = make(31, n, m, heads, kv, HD)
    given = (first, None if own else first_key, heads, kv, HD, scale, causal)
    got = run(dev, q, k, v, *given, kernel="fa_sequences_hd128")
    value, rng = sr.bf16_value(got).astype(np.float64), np.random.default_rng(0)
    for (a, b), (c, d) in zip(zip(first, first[1:]), zip(first_key, first_key[1:])):
        if a == b:
            continue
        at = sorted({0, b - a - 1, (b - a) // 2, min(63, b - a - 1), min(64, b - a - 1), *rng.integers(0, b - a, 8)})
        qf = sr.bf16_value(q[[a + i for i in at]]).astype(np.float64).reshape(len(at), heads, HD)
        kf, vf = (sr.bf16_value(x[c:d]).astype(np.float64).reshape(d - c, kv, HD) for x in (k, v))
        o, w, s = sr.softmax_rows(qf, kf, vf, scale, [max(0, i + 1 + (d - c) - (b - a)) if causal else d - c for i in at])
        sr.check(value[[a + i for i in at]].reshape(o.shape), (o, sr.bound(o, w, s, HD, True)), f"rows {at} of {a} .. {b}")
    # The longest sequence's last keys are not numbers (of a call without a limit: all of its keys, which the other sequences do not see)
    g = int(np.argmax(rows))
    length, count = first_key[g + 1] - first_key[g], rows[g]
    behind = min(length - 1, 150) if causal else length
    word = [0x7f80, 0xff80, 0x7fc0]
    for i in range(behind):
        k[first_key[g + 1] - 1 - i, i % 7::5] = word[i % 3]
        v[first_key[g + 1] - 1 - i, i % 5::3] = word[(i + 1) % 3]
    dirty = run(dev, q, k, v, *given, kernel="fa_sequences_hd128")
    untouched = np.ones(n, bool)
    untouched[first[g + 1] - min(behind, count):first[g + 1]] = False
    assert untouched.any() or len(rows) == 1 and not causal
    assert np.array_equal(dirty[untouched], got[untouched])
