"""Sources that ask for loads or stores with the streaming hint have such instructions in their compiled code: of a hinted and a plain access to one place behind
a test the compiler keeps the plain one, without a word (no GPU needed, hipcc only)."""
import os
import re

import pytest

from test_asm_hazards import CSRC, assembly, isa

SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))


@pytest.mark.parametrize("what", ["load", "store"])
@pytest.mark.parametrize("name", SOURCES)
def test_hints_are_in_the_compiled_code(name, what):
    code = re.sub(r"/\*.*?\*/|//[^\n]*", "", open(os.path.join(CSRC, name)).read(), flags=re.S)
    if f"__builtin_nontemporal_{what}" not in code:
        return
    assert any(l.startswith((f"global_{what}", f"buffer_{what}")) and re.search(r"\bnt\b", l) for l in isa(name))


def test_conversions_ask_for_it_on_values_of_two_bytes_alone():
    """A thread's 8 floats are two accesses of 16 bytes that share their lines with its neighbours': hinted, 4608 x 16384 of them took half as long again"""
    kernels = {l.split(":")[0] for l in assembly("mxfp4_ops.hip") if re.match(r"_Z\w*k_(to_mxfp4|mxfp4_to)I\w*:", l)}
    assert kernels and {k[-40:] for k in kernels if "If" in k and "Lb1" in k} == set()
    assert any("It" in k and "Lb1" in k for k in kernels)
