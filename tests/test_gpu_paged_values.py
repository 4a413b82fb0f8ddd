"""One-token attention over caches whose values are far from ordinary ones: rows whose scale says that they are not numbers."""
import numpy as np
import pytest

import sequences_reference as sr
from gpu_harness import Dev
from test_gpu_paged_cache import filled, rows

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
