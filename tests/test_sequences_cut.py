"""Which calls of packed attention have their keys cut into parts, and the search for how many blocks of keys make a part, by the function that the kernel
uses. Host arithmetic; no GPU."""
import os
import random
import subprocess

import pytest

import iris_c_amd
from test_half_words import CSRC, HIPCC, ROOT
from test_sequences_refusals import plan


@pytest.fixture(scope="module")
def lib():
    return iris_c_amd.load()


SPREAD = [round(200 * 80 ** random.Random(i).random()) for i in range(10)]


@pytest.mark.parametrize("rows,keys,heads,kv,cut", [
    ([16] * 32, [500] * 31 + [8000], 32, 8, True), ([16] * 32, [500] * 31 + [20000], 32, 8, True), ([16] * 32, [1024] * 32, 32, 8, True),
    ([100] * 10, SPREAD, 32, 8, True), ([100] * 10, SPREAD, 24, 24, True), ([16] * 32, [500] * 32, 32, 8, False), ([16] * 32, [2000] * 32, 24, 24, False),
    ([32], [16000], 32, 8, True), ([64, 1, 200, 17], [2064, 900, 4113, 1217], 32, 8, True), ([64], [900], 32, 8, True),
    ([64], [512], 32, 8, False)], ids=lambda v: str(v)[:24])
@pytest.mark.parametrize("causal", [0, 1])
def test_calls_that_are_cut(lib, rows, keys, heads, kv, cut, causal):
    """Those whose times stand beside the rule"""
    assert plan(lib, len(rows), sum(rows), sum(keys), heads, kv, causal, 0)[2] == (512 if cut else 1)


def test_the_search_for_the_blocks_of_a_part(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc here")
    program = str(tmp_path / "cut")
    r = subprocess.run([HIPCC, "-x", "hip", "-O2", "--offload-arch=gfx950", "-std=c++17", "-I" + CSRC, os.path.join(ROOT, "tests", "sequences_cut.cpp"), "-o", program],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([program], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout[-2000:]
    calls, searched, failed = (int(r.stdout.split("\n")[-2].split()[i]) for i in (0, 2, 4))
    assert calls > 10 ** 5 and searched > 10 ** 4 and failed == 0
