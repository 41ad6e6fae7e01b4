"""Wait states that inline assembly has to keep by itself.

The hardware wants an instruction between a scalar write of M0 and a load into LDS that takes its place from M0. The
compiler puts an s_nop 0 there for its own loads into LDS; it does not look into an asm statement.
"""
from __future__ import annotations

import re

import pytest

from aklr_amd import _build

SOURCES = sorted(p for p in _build.CSRC.rglob("*") if p.suffix in (".h", ".hip", ".cpp"))
WRITES_M0 = re.compile(r"s_\w+\s+m0\b")
INTO_LDS = re.compile(r"\blds\b")


def statements(text):
    """Instructions of each asm statement, in order."""
    for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(((?:\s*\"(?:[^\"\\]|\\.)*\")+)", text):
        template = "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1)))
        yield [line.strip() for line in re.split(r"\\n|;", template.replace("\\t", " ")) if line.strip()]


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_a_wait_state_between_m0_and_a_load_into_lds(path):
    for code in statements(path.read_text()):
        for before, after in zip(code, code[1:]):
            assert not (WRITES_M0.match(before) and INTO_LDS.search(after)), f"{before!r} right before {after!r}"
        if any(INTO_LDS.search(line) for line in code):  # the write belongs to the statement: what else runs before is not known
            assert any(WRITES_M0.match(line) for line in code), code


def test_the_statements_are_found():
    found = [code for path in SOURCES for code in statements(path.read_text())]
    assert sum(any(INTO_LDS.search(line) for line in code) for code in found) == 4
    assert list(statements('asm volatile("s_mov_b32 m0, %0\\n\\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(x));')) == [
        ["s_mov_b32 m0, %0", "buffer_load_dword %1, %2, 0 offen lds"]]
