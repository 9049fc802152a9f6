"""Buffer accesses that rely on their buffer's range to be dropped past its end keep the whole
offset where the range covers it: in the vector offset, with no register as scalar offset."""

import re

import pytest

from nanotitan_amd import build

SOURCES = sorted([*build.CSRC.glob("*.hip"), *build.CSRC.glob("*.hpp")])
# "buffer_load_dwordx4 %0, %1, <scalar offset> offen lds" in inline assembly
ACCESS = re.compile(r'"[^"\n]*\bbuffer_(?:load|store|atomic)\w*\s+([^"\n]*)"')


def test_the_accesses_are_found():
    text = 'asm("buffer_load_dwordx4 %0, %1, %2 offen lds")'
    assert ACCESS.findall(text) == ["%0, %1, %2 offen lds"]
    assert any(ACCESS.search(p.read_text()) for p in SOURCES)


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_no_scalar_offset(path):
    for operands in ACCESS.findall(path.read_text()):
        scalar = operands.split(",")[-1].split()[0]
        assert scalar == "0", operands
