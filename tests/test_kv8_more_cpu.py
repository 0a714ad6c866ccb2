"""Further refusals of the 8-bit cache's calls, without a GPU."""

import pytest

from redline_b200.ops.kernels import KernelError
from test_kv8_cpu import cache, prefill, write


def test_a_pool_without_a_page():
    """(page 0 is what a page id beyond the pool is read as)"""
    none = {n: t[:0].contiguous() for n, t in cache().items()}
    for call in (write, prefill):
        with pytest.raises(KernelError, match="without a page"):
            call(**none)
