"""The 64-bit form of MXFP4 that the GPU tests compare with, against the format's definition, and what the entries refuse (no GPU)."""
import ctypes as C

import numpy as np
import pytest

import mxfp4_reference as mx

_vp = C.c_void_p


def test_every_code_and_scale_comes_back():
    halves = np.arange(16, dtype=np.uint8)
    codes = np.zeros((1, 16), np.uint8)
    codes[0, :8] = halves[0::2] | halves[1::2] << 4
    for s in (0, 1, 126, 127, 128, 252, 253):
        v = mx.decode(codes, np.array([[s]], np.uint8), 32)
        assert np.array_equal(v[0, :16] * 2.0 ** (127 - s), [0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])
        if 0 < s < 253:                                        # 6 X and 2 X: the block's own scale again
            c, t = mx.encode(v.astype(np.float32))
            assert t[0, 0] == s and np.array_equal(c, codes)
    assert np.isnan(mx.decode(codes, np.array([[255]], np.uint8), 32)).all()


def test_ties_go_to_the_even_code_and_large_values_to_six():
    x = np.zeros((1, 32), np.float32)
    x[0, :12] = [4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7.99, -.25, -5, -7]
    c, s = mx.encode(x)
    assert s[0, 0] == 127
    assert np.array_equal(mx.decode(c, s, 12)[0], [4, 0, 1, 1, 2, 2, 4, 4, 6, 0, -4, -6])


def test_a_value_is_off_by_half_a_step_at_most():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((64, 100)) * np.exp2(rng.integers(-120, 120, (64, 1)))).astype(np.float32)
    c, s = mx.encode(x)
    y = mx.decode(c, s, 100)
    scale = np.repeat(np.exp2(s.astype(np.float64) - 127), 32, 1)[:, :100]
    r = np.abs(x) / scale
    assert (r < 8).all()
    step = np.where(r < 2, .5, np.where(r < 4, 1, 2))
    assert (np.abs(y - x)[r <= 6] <= (step * scale / 2)[r <= 6]).all()
    assert (np.abs(y)[r > 6] == 6 * scale[r > 6]).all()


def test_extremes():
    x = np.zeros((6, 32), np.float32)
    x[1, 0], x[2, 0], x[3, 0] = 1e-45, np.float32(2.0 ** -125), np.finfo(np.float32).max
    x[4, 3], x[5, 7] = np.inf, np.nan
    c, s = mx.encode(x)
    assert s[:, 0].tolist() == [0, 0, 0, 252, 255, 255]
    assert mx.decode(c, s, 32)[3, 0] == 6 * 2.0 ** 125 and not c[4:].any()


@pytest.fixture(scope="module")
def lib():
    import os

    import iris_c_amd
    if not os.path.exists(iris_c_amd.LIB_PATH):
        iris_c_amd.build()
    return iris_c_amd.load()


P, ODD = 1 << 20, (1 << 20) + 8                                   # never read: every call here ends at its arguments

REFUSED = [
    ("f32_to_mxfp4", (None, P, P, 8, 2, 8), "missing"),
    ("f32_to_mxfp4", (P, None, P, 8, 2, 8), "missing"),
    ("bf16_to_mxfp4", (P, P, None, 8, 2, 8), "missing"),
    ("bf16_to_mxfp4", (P, P, P, 7, 2, 8), "ld >= cols"),
    ("f32_to_mxfp4", (P, P, P, -8, 2, 8), "ld >= cols"),
    ("f32_to_mxfp4", (ODD, P, P, 8, 2, 8), "aligned"),
    ("mxfp4_to_f32", (P, 7, P, P, 2, 8), "ld >= cols"),
    ("mxfp4_to_bf16", (None, 8, P, P, 2, 8), "missing"),
    ("mxfp4_to_bf16", (P, 8, ODD, P, 2, 8), "aligned"),
    ("linear_mxfp4_f32", (P, P, P, P, P, 4, 0, 4), "positive"),
    ("linear_mxfp4_bf16", (P, P, P, P, P, 4, -3, 4), "positive"),
    ("linear_mxfp4_f32", (None, P, P, P, P, 4, 8, 4), "missing"),
    ("linear_mxfp4_f32", (P, P, None, P, P, 4, 8, 4), "missing"),
    ("linear_mxfp4_bf16", (P, P, P, P, None, 4, 8, 4), "missing"),
    ("linear_mxfp4_bf16", (P, ODD, P, P, P, 4, 8, 4), "aligned"),
    ("linear_mxfp4_bf16", (P, P, P, ODD, P, 4, 8, 4), "aligned"),
    ("linear_mxfp4_f32_grouped", (P, P, P, P, P, None, 2, 4, 8, 4), "first rows"),
    ("linear_mxfp4_bf16_grouped", (P, P, P, P, P, P, -1, 4, 8, 4), "first rows"),
    ("linear_mxfp4_bf16_grouped", (P, P, P, ODD, P, P, 2, 4, 8, 4), "aligned"),
    ("linear_mxfp4_f32_grouped", (P, P, P, P, P, P, 2, 4, 0, 4), "positive"),
    ("linear_f32_grouped", (P, P, P, None, 2, 4, 8, 4), "first rows"),
    ("linear_bf16_grouped", (P, P, P, P, -1, 4, 8, 4), "first rows"),
    ("linear_bf16_grouped", (P, P, P, P, 2, 4, 0, 4), "positive"),
    ("linear_bf16_grouped", (P, None, P, P, 2, 4, 8, 4), "missing"),
]


@pytest.mark.parametrize("name,args,said", REFUSED)
def test_refused_calls_say_why(lib, capfd, name, args, said):
    lib.iris_dev_last_error()
    getattr(lib, "iris_dev_" + name)(*args)
    assert lib.iris_dev_last_error() != 0
    assert said in capfd.readouterr().err


EMPTY = [
    ("f32_to_mxfp4", (P, P, P, 8, 0, 8)), ("bf16_to_mxfp4", (P, P, P, 8, 4, 0)), ("mxfp4_to_f32", (P, 8, P, P, 0, 8)), ("mxfp4_to_bf16", (P, 8, P, P, -1, 8)),
    ("linear_mxfp4_f32", (P, P, P, P, P, 0, 8, 4)), ("linear_mxfp4_bf16", (P, P, P, P, P, 4, 8, 0)),
    ("linear_mxfp4_f32_grouped", (P, P, P, P, P, P, 0, 4, 8, 4)), ("linear_mxfp4_bf16_grouped", (P, P, P, P, P, P, 2, 0, 8, 4)),
    ("linear_f32_grouped", (P, P, P, P, 0, 4, 8, 4)), ("linear_bf16_grouped", (P, P, P, P, 2, 4, 8, 0)),
]


@pytest.mark.parametrize("name,args", EMPTY)
def test_calls_with_nothing_to_do_do_nothing(lib, name, args):
    lib.iris_dev_last_error()
    getattr(lib, "iris_dev_" + name)(*args)
    assert lib.iris_dev_last_error() == 0


def test_no_device_no_answer(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for name, args in [("f32_to_mxfp4", (P, P, P, 8, 2, 8)), ("mxfp4_to_bf16", (P, 8, P, P, 2, 8)), ("linear_mxfp4_f32", (P, P, P, P, P, 4, 8, 4)),
                       ("linear_mxfp4_bf16_grouped", (P, P, P, P, P, P, 2, 4, 8, 4)), ("linear_f32_grouped", (P, P, P, P, 2, 4, 8, 4))]:
        lib.iris_dev_last_error()
        getattr(lib, "iris_dev_" + name)(*args)
        assert lib.iris_dev_last_error() != 0, name
