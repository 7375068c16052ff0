"""Registers that inline assembly may not write behind the compiler's back."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "aegaeon_amd" / "csrc"


def test_the_compiler_sets_m0():
    """m0 is reserved: a clobber list cannot give it away, and the compiler sets it for
    instructions of its own. Assembly takes it as an input ("{m0}") and does not write it."""
    found = []
    for path in sorted((*CSRC.glob("*.h"), *CSRC.glob("*.hip"))):
        for m in re.finditer(r"\basm\b[^;]*;", path.read_text()):
            text = m[0]
            takes = '"{m0}"' in text
            if re.search(r"\bs_\w+ m0\b", text) or ("_lds_" in text and not takes):
                found.append((path.name, " ".join(text.split())[:80]))
    assert not found, found
