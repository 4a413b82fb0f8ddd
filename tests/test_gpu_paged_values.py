"""One-token attention over caches whose values are far from ordinary ones: rows whose scale says that they are not numbers, huge values that have no
weight, values next to zero."""
import numpy as np
import pytest

import sequences_reference as sr
from gpu_harness import Dev
from test_gpu_paged_cache import KINDS, filled, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


@pytest.mark.parametrize("hd", [128, 96])
@pytest.mark.parametrize("which", ["ks", "vs"])
@pytest.mark.parametrize("length", [60, 3000])
def test_a_scale_of_255_is_not_a_number_whatever_the_codes(dev, length, which, hd):
    """In a cache that another program filled: byte 255 over ordinary codes, over zeros and over codes that are NaN themselves"""
    kv, heads, lengths = 2, 4, [50, length, 40]
    c = filled(dev, "fp8", lengths, 16, kv, hd)
    q = rows(3, 3, heads * hd)
    clean = c.attend(lengths, q, heads, hd ** -0.5)
    bytes_, codes = getattr(c, which), getattr(c, which[0])
    (page0, at0), (page1, at1), (page2, at2) = c.place(1, length - 1), c.place(0, 7), c.place(2, 0)
    bytes_[page0, 1, at0] = bytes_[page1, 0, at1] = bytes_[page2, 1, at2] = 255
    codes[page1, 0, at1], codes[page2, 1, at2] = 0, 0x7f
    for d, a in ((getattr(c, "d" + which), bytes_), (getattr(c, "d" + which[0]), codes)):
        dev.lib.iris_dev_upload(d, a.ctypes.data, a.nbytes)
    got = c.attend(lengths, q, heads, hd ** -0.5, compare=False, kernel="fa_paged_hd128" if hd == 128 else "attention_paged_generic")
    bad = np.zeros((3, kv, heads // kv * hd), bool)
    bad[1, 1] = bad[0, 0] = bad[2, 1] = True
    bad = bad.reshape(3, -1)
    assert np.isnan(sr.bf16_value(got[bad])).all()
    assert np.array_equal(got[~bad], clean[~bad])
    c.read(lengths, sum(lengths), np.concatenate([[0], np.cumsum(lengths)]))
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("length,at", [(20, 0), (20, 19), (70, 33), (1500, 0), (1500, 1499), (1500, 700)])
def test_a_huge_value_without_weight_has_no_part(dev, kind, length, at):
    """Its score lies 362 below the others': exp of that is nothing in 32 bits, and 10^-157 in 64"""
    kv, heads, hd = 1, 4, 128
    c = filled(dev, kind, [length], 16, kv, hd)
    k, v = np.full((length, hd), 4.0, np.float32), sr.bf16_value(rows(5, length, hd)).copy()
    k[at], v[at] = -4.0, 3e38
    c.write([length], sr.bf16_round(k), sr.bf16_round(v), [0, length])
    c.attend([length], sr.bf16_round(np.full((1, heads * hd), 4.0, np.float32)), heads, hd ** -0.5, kernel="fa_paged_hd128")
    dev.free_all()


@pytest.mark.parametrize("exponent", [-100, -110, -116, -120, -126, -132])
@pytest.mark.parametrize("length", [3, 300])
def test_values_next_to_zero(dev, length, exponent):
    """Rows of V whose scales are 2^(exponent - 7) and thereabouts, down to the least there is"""
    kv, heads, hd = 2, 8, 128
    c = filled(dev, "fp8", [length], 16, kv, hd)
    v = np.ldexp(sr.bf16_value(rows(6, length, kv * hd)), exponent).astype(np.float32)
    c.write([length], rows(7, length, kv * hd), sr.bf16_round(v), [0, length])
    c.attend([length], rows(8, 1, heads * hd), heads, hd ** -0.5, kernel="fa_paged_hd128")
    dev.free_all()
