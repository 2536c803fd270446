"""What the HIP sources have to say to the compiler, read from their text."""

from __future__ import annotations

import re

import pytest

from .conftest import REPO_ROOT

SOURCES = sorted((REPO_ROOT / "exl3_intel_arc_quantizer_amd" / "csrc").glob("*.h*"))


def _statements(text: str) -> list:
    """The inline assembly of a source, each with its operands and clobbers."""
    return re.findall(r"\basm\s+volatile\s*\((.*?)\);", text, re.S)


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_assembly_names_the_registers_it_writes(source):
    """Registers that the text writes by name are named as clobbered, so that the
    compiler holds nothing in them."""
    for statement in _statements(source.read_text()):
        parts = statement.split('"')
        code, clobbers = "".join(parts[1:2]), statement.rsplit(":", 1)[-1]
        for register in re.findall(r"\bs_mov_b32\s+(m0|s\d+|vcc_lo|vcc_hi|exec_lo|exec_hi)\b", code):
            assert f'"{register}"' in clobbers, (source.name, statement)
