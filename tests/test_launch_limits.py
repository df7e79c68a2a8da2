"""A launch of more threads than a dimension takes is refused before HIP sees it, which would launch a part of them.  No GPU."""
import ctypes

import pytest

INVALID_CONFIGURATION = 9  # hipErrorInvalidConfiguration


# 8 elements to a thread: 2^32 threads and more
@pytest.mark.parametrize("elements", [1 << 35, (1 << 35) + 12345, 1 << 37])
def test_add(elements):
    import llm_simple_amd.ops as ops
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) & ~15  # (nothing is launched that would look there)
    assert ops.lib.llmhip_add(p, p, p, elements, 5, None) == INVALID_CONFIGURATION
