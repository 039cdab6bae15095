"""How the kernels' clusters meet, read from their sources: a block whose shared memory others read may leave only when they have read it, and what
tells it so is an arrival that orders the reads before it."""

import re
from pathlib import Path

import pytest

from lalamo_b200 import native

SOURCES = sorted(Path(native.source_files()[0]).parent.glob("*.cu*"))


def code_of(path):
    return re.sub(r"//[^\n]*", "", path.read_text())


@pytest.mark.parametrize("path", SOURCES, ids=lambda path: path.name)
def test_arrivals_order_what_was_read(path):
    """``.relaxed`` orders nothing: a block could leave, and its shared memory go to another, while a read of it is under way."""
    arrivals = re.findall(r"barrier\.cluster\.arrive[.\w]*", code_of(path))
    assert all(".release" in arrival for arrival in arrivals), arrivals
    waits = re.findall(r"barrier\.cluster\.wait[.\w]*", code_of(path))
    assert all(".acquire" in wait for wait in waits), waits


def test_there_are_meetings():
    assert any("barrier.cluster.arrive" in code_of(path) for path in SOURCES)


def test_warps_that_may_have_parted_meet_first():
    """The aligned forms want a warp's lanes together; behind writes that only some lanes make they may not be."""
    code = code_of(next(path for path in SOURCES if path.name == "gemm_microscaled.cu"))
    found = [match.start() for match in re.finditer(r'asm volatile\("barrier\.cluster\.(arrive|wait)', code)]
    assert len(found) == 2
    for place in found:
        assert "__syncwarp();" in code[place - 120 : place]
