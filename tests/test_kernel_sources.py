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


@pytest.mark.parametrize("name,entry", [("dense.cu", "t2sc_dense_linear_device"), ("rope.cu", "t2sc_rope_apply_device"),
                                        ("rope.cu", "t2sc_qk_norm_rope_device"), ("attention.cu", "t2sc_attention_device")])
def test_a_wait_that_gave_up_reaches_the_next_call(name, entry):
    """The attention block's kernels follow torch's streams and need not be synchronised through their context: they note a wait
    that gave up in host memory (the device self-test checks the way there), and each operator reports it before it launches."""
    text = open(os.path.join(CSRC, name)).read()
    body = text[text.index(f"int {entry}("):]
    body = body[:body.index("\n}\n")]
    assert body.index("T2SC_TRY(earlier_failure(ctx))") < body.index("DeviceGuard")


@pytest.mark.parametrize("name", [f for f in SOURCES if f != "rope.cu" and f != "dense_rows.cu"])
def test_bounded_waits_report_into_host_memory(name):
    """(rope.cu and dense_rows.cu wait for nothing.)"""
    assert "ctx->d_wait" in SOURCES[name] and "d_err" not in SOURCES[name]
