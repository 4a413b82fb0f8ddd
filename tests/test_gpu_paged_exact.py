"""One-token attention on the matrix cores is as exact as its own rounding: P goes in two bf16 parts, Q against 8-bit keys in two parts of 4 bits. Held to that
in short and long texts, finished by one wave and joined from the parts of many."""
import ctypes as C

import numpy as np
import pytest

import sequences_reference as sr
from gpu_harness import Dev
from test_gpu_paged_cache import filled, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


def half_step(x):
    """of bf16, at |x|"""
    return np.ldexp(1.0, np.frexp(np.maximum(x, 2.0 ** -126))[1] - 9)


def tight(out, weight, size, hd, scores, adds):
    """The output's rounding; the rest of P, less than 2^-7 of it, rounded by half a step of 2^-8 at most, and its last bit; twice what a score may be off by
    because of Q's parts (above and below the line); f32 arithmetic as in sequences_reference.bound, and `adds` further sums."""
    off = (2.0 ** -15 + 2.0 ** -23 + 2 * scores + (2 * (hd + 8) * size + 64 + adds) * 2.0 ** -24) * weight
    return half_step(np.abs(out) + off) + off * (1 + sr.HALF) + 2.0 ** -126


CASES = {
    # lengths, query heads, kv heads, further columns of the table, threads that join
    "short": ([1, 17, 0, 31, 33, 90], 8, 2, 0, 256), "ordinary": ([700, 3, 0, 129, 1030], 32, 8, 0, 256), "no group": ([257, 400], 5, 5, 0, 256),
    "one long": ([20011], 8, 1, 0, 512), "two long": ([5000, 12003], 16, 2, 0, 512), "a long one among short ones": ([5, 9001, 0, 77], 8, 2, 0, 256),
    "two blocks of heads": ([24001], 17, 1, 0, 512), "a wide table": ([300], 32, 8, 9000, 256), "a wide table, one head": ([300, 1], 1, 1, 9000, 512),
    "one wave": ([16], 3, 1, 0, 0),
}


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_as_exact_as_its_rounding(dev, case, kind):
    lengths, heads, kv, more, join = CASES[case]
    hd, page, fp8 = 128, 16, kind == "fp8"
    c = filled(dev, kind, lengths, page, kv, hd, seed=21, extra_columns=more)
    waves, threads = C.c_int(), C.c_int()
    dev.lib.iris_hip_paged_plan(int(fp8), 4, c.table.shape[1], len(lengths), heads, kv, C.byref(waves), C.byref(threads))
    assert threads.value == join
    q, scale, values = rows(23, len(lengths), heads * hd, 1.3), hd ** -0.5, c.values()
    got = c.attend(lengths, q, heads, scale, kernel="fa_paged_hd128", compare=False)
    tiles = sum(-(-n // (64 if fp8 else 32)) for n in lengths) * kv * -(-heads // kv // 16)
    adds = 4 * -(-tiles // waves.value) + max(lengths) / 32
    for g, n in enumerate(lengths):
        o, w, s = sr.softmax_rows(*(x for x in qkv(c, values, q[g], g, n, heads)), scale, [n])
        # Q's second part is exact down to a step of 2^-9 of its scale, of which the column's largest value is more than 224
        k = np.abs(qkv(c, values, q[g], g, n, heads)[1]).sum(-1).max(initial=0.0)
        scores = 2.0 ** -10 / 224 * np.abs(sr.bf16_value(q[g])).reshape(1, heads, hd).max(-1, keepdims=True).astype(np.float64) * k * scale if fp8 else 0.0
        sr.check(sr.bf16_value(got[g]).astype(np.float64).reshape(o.shape), (o, tight(o, w, s, hd, scores, adds)), f"sequence {g}")
    dev.free_all()


def qkv(c, values, q, g, n, heads):
    at = np.arange(n)
    page, place = c.table[g, at // c.page], at % c.page
    return sr.bf16_value(q).astype(np.float64).reshape(1, heads, c.hd), values[0][page, :, place], values[1][page, :, place]
