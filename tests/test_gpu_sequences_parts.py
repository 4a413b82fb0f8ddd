"""Packed attention where the keys of a workgroup are cut into parts: what is not a number on both sides of a part's end, seen by some rows and not by
others."""
import numpy as np
import pytest

import sequences_reference as sr
from gpu_harness import Dev
from test_gpu_sequences import make, parts, reference, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


@pytest.mark.parametrize("behind", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 2)])
@pytest.mark.parametrize("keys", [2109, 2125, 2320])
def test_limits_on_both_sides_of_a_parts_end(dev, keys, heads, kv, behind):
    """90 rows. The last part holds the last block of keys alone (2109: block 32, 2320: block 36), and the limits of one wave's columns lie in it and in the
    block in front. Infinities, each in a dim of its own, at the limits of every third row; in dim 127 a value that only the last four rows see: those
    in front have nothing of it, and their infinities stay what they are."""
    n, hd = 90, 128
    assert parts(dev, 1, n, keys, heads, kv, True) > 1
    q, k, v = make(11, n, keys, heads, kv, hd)
    clean = v.copy()
    at = {d: 3 * d for d in range(29)}
    for h in range(kv):
        for d, i in at.items():
            v[keys - n + i, hd * h + d] = 0xff80 if d % 2 else 0x7f80
            clean[keys - n + i, hd * h + d] = 0
        v[keys - 4, hd * h + 127] = sr.bf16_round(np.float32(behind))
        clean[keys - 4, hd * h + 127] = 0
    got = run(dev, q, k, v, [0, n], [0, keys], heads, kv, hd, hd ** -0.5, True, kernel="fa_sequences_hd128")
    want, limit = reference(q, k, clean, [0, n], [0, keys], heads, kv, hd, hd ** -0.5, True, True)
    have = sr.bf16_value(got).astype(np.float64)
    for h in range(heads):
        for d, i in at.items():
            c = hd * h + d
            assert np.isfinite(have[:i, c]).all() and (have[i:, c] == (-np.inf if d % 2 else np.inf)).all(), (h, d, have[i:, c])
            have[i:, c] = want[i:, c] = 0
        c = hd * h + 127
        last = have[n - 4:, c]
        assert np.isnan(last).all() if np.isnan(behind) else (last == behind).all()
        have[n - 4:, c] = want[n - 4:, c] = 0
    sr.check(have, (want, limit))
