"""Sources that ask for loads or stores with the streaming hint have such instructions in their compiled code: of a hinted and a plain access to one place behind
a test the compiler keeps the plain one, without a word (no GPU needed, hipcc only)."""
import os
import re

import pytest

from test_asm_hazards import CSRC, isa

SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))


@pytest.mark.parametrize("what", ["load", "store"])
@pytest.mark.parametrize("name", SOURCES)
def test_hints_are_in_the_compiled_code(name, what):
    code = re.sub(r"/\*.*?\*/|//[^\n]*", "", open(os.path.join(CSRC, name)).read(), flags=re.S)
    if f"__builtin_nontemporal_{what}" not in code:
        return
    assert any(l.startswith((f"global_{what}", f"buffer_{what}")) and re.search(r"\bnt\b", l) for l in isa(name))
