"""An infinity in V that a row sees, its key's score far below or above the row's others: that infinity in its dim while the score is not more than 70 below the
largest, that or NaN beyond, and nothing in any other dim; in every order of the keys, in short and long texts, cut and whole."""
import numpy as np
import pytest

import sequences_reference as sr
from gpu_harness import Dev
from test_gpu_paged_cache import filled
from test_gpu_paged_cache import rows as random_rows
from test_gpu_sequences import run

pytestmark = pytest.mark.gpu
DIM = 5


@pytest.fixture(scope="module")
def dev():
    return Dev()


def keys(n, at, hd, below):
    """K whose rows score 45 with q, but row `at`, which scores `below` less (against rows of 4 of as many dims, scale hd ** -0.5); and V"""
    k = np.ones((n, hd), np.float32)
    k[at] = 1.0 - below / (4.0 * hd ** 0.5)
    v = random_rows(3, n, hd)
    return sr.bf16_round(k), v


def check(got, clean, sees, below):
    got, clean = sr.bf16_value(got), sr.bf16_value(clean)
    there = got[sees][:, :, DIM]
    assert (there == np.inf).all() if below <= 70 else (np.isnan(there) | (there == np.inf)).all(), there
    got[sees, :, DIM] = clean[sees, :, DIM] = 0.0
    assert np.isfinite(got).all() and np.array_equal(got, clean)


@pytest.mark.parametrize("below", [-60, 0, 20, 70, 120, 400])
@pytest.mark.parametrize("n,at", [(20, 0), (20, 19), (70, 3), (70, 40), (1500, 0), (1500, 750), (1500, 1499)])
@pytest.mark.parametrize("hd", [128, 96])
def test_one_token(dev, n, at, below, hd):
    heads = 4
    c = filled(dev, "bf16", [n], 16, 1, hd)
    k, v = keys(n, at, hd, below)
    q = sr.bf16_round(np.full((1, heads * hd), 4.0, np.float32))
    out = []
    for value in (0, 0x7f80):
        v[at, DIM] = value
        c.write([n], k, v, [0, n])
        out.append(c.attend([n], q, heads, hd ** -0.5, compare=False, kernel="fa_paged_hd128" if hd == 128 else "attention_paged_generic").reshape(1, heads, hd))
    check(out[1], out[0], np.array([True]), below)
    dev.free_all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("below", [-60, 0, 20, 70, 120, 400])
@pytest.mark.parametrize("m,at", [(100, 0), (100, 63), (100, 64), (100, 99), (2109, 5), (2109, 1000), (2109, 2030), (2109, 2100)])
@pytest.mark.parametrize("hd", [128, 96])
def test_packed_rows(dev, m, at, below, causal, hd):
    """90 rows; over 2109 keys they are cut into parts"""
    n, heads = 90, 2
    k, v = keys(m, at, hd, below)
    q = sr.bf16_round(np.full((n, heads * hd), 4.0, np.float32))
    out = []
    for value in (0, 0x7f80):
        v[at, DIM] = value
        out.append(run(dev, q, k, v, [0, n], [0, m], heads, 1, hd, hd ** -0.5, causal,
                       kernel="fa_sequences_hd128" if hd == 128 else "attention_sequences_generic").reshape(n, heads, hd))
    check(out[1], out[0], np.arange(n) + 1 + m - n > at if causal else np.ones(n, bool), below)
