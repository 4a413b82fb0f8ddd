"""Rows that start in the middle of 4 bytes are read in whole words: none of the reads leaves its matrix, whatever the matrix starts
at. The addresses are computed on the host by the functions that the kernel uses; no GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "iris_c_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def test_no_word_is_read_outside_its_matrix(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc here")
    program = str(tmp_path / "reads")
    r = subprocess.run([HIPCC, "-x", "hip", "-O2", "--offload-arch=gfx950", "-std=c++17", "-I" + CSRC, os.path.join(ROOT, "tests", "half_words_reads.cpp"),
                        "-o", program], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([program], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[-2000:]
    reads, outside = r.stdout.split()[0], r.stdout.split()[2]
    assert int(reads) > 10 ** 5 and int(outside) == 0
