"""Rules that the kernels keep in their sources, where breaking one would hang
or race on a GPU instead of failing."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "trellis2-mojo_b200", "csrc")


def _sources():
    found = {}
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        if "next_kernel_may_start" in text or "launch_overlapped" in text:
            found[os.path.basename(path)] = text
    return found


SOURCES = _sources()
ALLOCATING = [f for f, text in SOURCES.items() if "tmem_alloc" in text]


def test_the_overlapped_kernels_are_found():
    assert len(SOURCES) >= 5 and len(ALLOCATING) >= 3


@pytest.mark.parametrize("name", ALLOCATING)
def test_tensor_memory_is_allocated_before_the_next_kernel_may_start(name):
    """The next kernel's blocks hold the tensor memory that they allocate until this kernel has ended: a block of this one that
    allocates after letting them start could wait for ever. The allocation is one warp's, so a barrier of the block (of the
    pair, where the pair allocates) stands between the two."""
    text = SOURCES[name]
    starts = [m.start() for m in re.finditer(r"next_kernel_may_start\(\)", text)]
    assert len(starts) == 1
    last = max(m.end() for m in re.finditer(r"tmem_alloc(_pair)?\(", text))
    assert last < starts[0]
    between = text[last:starts[0]]
    assert "__syncthreads()" in between
    if "tmem_alloc_pair" in text:
        assert "cluster_sync()" in between


@pytest.mark.parametrize("name", SOURCES)
def test_non_coherent_loads_are_of_the_handles_own_tables(name):
    """__ldg needs memory that nothing writes during the kernel's whole life. An overlapped kernel's life begins while the one
    before it writes, so rows, weights, gains, biases and coordinates are read by ordinary loads."""
    text = SOURCES[name]
    asked = [re.match(r"\s*(reinterpret_cast<[^>]*>\()?\s*([\w.]+)", text[m.end():]).group(2)
             for m in re.finditer(r"\b__ldg\(", text)]
    assert set(asked) <= {"a.seqs", "a.blocks", "a.turns"}, asked
