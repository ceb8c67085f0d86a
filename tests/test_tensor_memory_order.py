"""When the kernels of the library take tensor memory, read from their sources.

The allocation of tensor memory waits, without a bound, until the multiprocessor has the columns.  So a kernel on block-scaled
products takes them after its dependency wait, when no kernel before it in the stream can still want any.
"""

import os
import re

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
