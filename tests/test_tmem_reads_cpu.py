"""Registers of a TMEM load are undefined until its wait, and the compiler does not know: plain arithmetic on them may be
moved in front of a wait that names only memory. So each load's registers pass through an asm statement behind the
wait (``reg_fence32`` or one with "+r" operands), or load and wait are one statement. Checked in the sources, as a build
that happens to keep the order shows nothing."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "taomate-h3_b200" / "csrc"
SOURCES = sorted(p.name for p in [*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")] if "tcgen05.ld" in p.read_text() or "tmem_ld" in p.read_text())


def _statement(text: str, at: int) -> str:
    return text[at:text.index(";\n", at)]


def test_there_are_sources() -> None:
    assert "h3sa_ptx.cuh" in SOURCES and "h3sa_branch.cu" in SOURCES


@pytest.mark.parametrize("name", SOURCES)
def test_loads_are_tied_to_their_waits(name) -> None:
    text = (CSRC / name).read_text()
    for m in re.finditer(r"asm volatile\(", text):  # helpers that return what they load have waited for it
        asm = _statement(text, m.start())
        if "tcgen05.ld." in asm and "return" in text[m.start() + len(asm):m.start() + len(asm) + 20]:
            assert "tcgen05.wait::ld" in asm, asm
    for m in re.finditer(r"(?<!void )\btmem_ld(16|32)\(", text):
        wait = text.find("tmem_wait_ld();", m.start())
        assert 0 <= wait - m.start() < 400, text[m.start():m.start() + 80]
        behind = text[wait:wait + 220]
        assert "reg_fence32(" in behind or '"+r"' in behind, text[m.start():m.start() + 80]
