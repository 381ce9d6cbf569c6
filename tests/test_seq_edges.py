"""Sequence operators without a GPU: what the sources promise the compiler, and
refusals at the edges of arguments and layouts."""
from __future__ import annotations

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "cusr_amd" / "csrc"


# -------------------------------------------------------------------- sources

def test_assembly_names_what_it_overwrites():
    """Assembly that writes m0 says so: the compiler may keep a value there."""
    found = 0
    for path in sorted(CSRC.glob("seq_*")):
        for block in re.findall(r"asm volatile\((.*?)\);", path.read_text(), re.S):
            if re.search(r"s_mov_b32 m0", block):
                found += 1
                clobbers = block.rsplit(":", 1)[1]
                assert '"m0"' in clobbers and '"memory"' in clobbers, (path.name, block)
    assert found >= 3
