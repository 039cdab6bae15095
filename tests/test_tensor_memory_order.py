"""The order in which kernels get tensor memory, read from their sources.  A CTA waits for tensor memory without a limit, and one that starts early may hold some while it waits for
the kernel before it.  So no kernel lets its successor start before it has its own, unless its CTAs leave no room beside them for another that uses some: then nobody
who holds tensor memory waits for somebody who wants some."""

import re
from pathlib import Path

import pytest

from lalamo_b200 import native

# bytes of shared memory that no kernel with tensor memory does without, what a multiprocessor has, and what it keeps for each CTA
LEAST, WHOLE, RESERVED = 16 << 10, 228 << 10, 1 << 10
# shared memory of the kernels that let their successor start before they have tensor memory
ALONE = {"gemm_tcgen05_persistent_kernel": 4 * 48 * 1024 + 2 * 16 * 1024 + 1024 + 256, "moe_tcgen05_kernel": 1024 + 196608 + 2 * 128 * 80 + 2 * 1025 * 4}


def kernels():
    """Name and body of every kernel that allocates tensor memory."""
    found = []
    for path in sorted(Path(native.source_files()[0]).parent.glob("*.cu*")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        starts = [match.start() for match in re.finditer(r"__global__", text)] + [len(text)]
        for begin, end in zip(starts, starts[1:]):
            body = text[begin:end]
            if "tcgen05.alloc" in body:
                found.append((re.search(r"(\w+)\s*\(const", body).group(1), body))
    return found


def test_the_kernels_are_found():
    names = {name for name, _ in kernels()}
    assert {"gemm_tcgen05_kernel", "gemm_microscaled_kernel", "gemm_microscaled_split_kernel", "attention_tcgen05_kernel"} | set(ALONE) <= names


@pytest.mark.parametrize("name,body", kernels(), ids=lambda value: value if len(value) < 64 else "")
def test_successors_start_behind_the_allocation(name, body):
    if name in ALONE:
        assert WHOLE - 2 * RESERVED - ALONE[name] < LEAST
        return
    allowed = [match.start() for match in re.finditer(r"allow_next_kernel\(\)", body)]
    assert allowed and min(allowed) > max(match.start() for match in re.finditer(r"tcgen05\.alloc", body))


def test_the_sizes_are_the_sources():
    folder = Path(native.source_files()[0]).parent
    assert "kPersistSharedBytes = 4 * 48 * 1024 + kPersistExchangeBytes + 1024 + 256" in (folder / "gemm_tcgen05.cu").read_text()
    moe = (folder / "moe_tcgen05.cu").read_text()
    assert "kMoeStageArea = 196608" in moe and "kMoePitch = 80" in moe and "most = 1024 + kMoeStageArea + 2 * kMoeRows * kMoePitch + 2 * (kMoeMaxExperts + 1) * 4" in moe


def test_loads_of_tensor_memory_hold_their_wait():
    """What a load of sixteen columns brings is there when its statement ends: with the wait in a statement of its own, whatever only uses the values may be placed between the two."""
    text = (Path(native.source_files()[0]).parent / "tcgen05.cuh").read_text()
    body = text[text.index("void tmem_load_16(") :]
    body = body[: body.index("\n}")]
    assert body.count("asm volatile") == 1 and body.index("tcgen05.ld.") < body.index("tcgen05.wait::ld")
