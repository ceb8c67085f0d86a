"""When the kernels of the library take tensor memory, read from their sources.

The allocation of tensor memory waits, without a bound, until the multiprocessor has the columns.  So a kernel on block-scaled
products takes them after its dependency wait, when no kernel before it in the stream can still want any, and a kernel on pairs of
multiprocessors, which holds all of theirs, is launched in plain stream order and lets nothing be scheduled under it.
"""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "thing_htn_2026_b200", "csrc")


def code(name):
    """A source file without its comments."""
    with open(os.path.join(CSRC, name)) as handle:
        text = handle.read()
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", text, flags=re.S))


def kernel(name, which):
    """The text of a kernel, up to what follows it at the margin."""
    text = code(name)
    at = re.search(rf"__global__[^;{{]*\b{which}\(", text).start()
    return text[at:text.index("\n}\n", at)]


def test_few_rows_take_tensor_memory_after_the_kernels_before():
    text = kernel("mx4_stream.cu", "mx4_stream_kernel")
    branch = text[text.index("warp == 1"):]
    assert 0 <= branch.find("pdl_wait()") < branch.index("tcgen05.alloc")


@pytest.mark.parametrize("name,which", [("mx4_pair.cu", "mx4_pair_kernel"), ("moe_grouped.cu", "pair_gemm_kernel")])
def test_pairs_run_alone_and_leave_together(name, which):
    text = kernel(name, which)
    assert "cta_group::2" in text and "pdl_launch_dependents" not in text
    # the cluster barrier counts threads: the warps' lanes may come apart ahead of it
    assert "barrier.cluster" in code(name) and not re.search(r"barrier\.cluster\.\w+\.aligned", code(name))
    # behind the release of the pair's columns both blocks meet once more
    assert "pair_barrier();" in text[text.index("tcgen05.dealloc"):]
    # a whole warp, its lanes together, takes and releases them
    for place in ("tcgen05.alloc", "tcgen05.dealloc"):
        before = text[:text.index(place)]
        assert before.rindex("__syncwarp()") > before.rindex("if (threadIdx.x == 0)" if place == "tcgen05.alloc" else "pair_barrier()")
    launches = re.findall(r"(thn_launch\w*)\(kernel,", code(name))
    assert launches == ["thn_launch_ordered"]
