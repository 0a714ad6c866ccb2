"""Further refusals of the 8-bit cache's calls, without a GPU."""

import ctypes

import pytest

from redline_b200.ops import kernels
from redline_b200.ops.kernels import KernelError
from test_kv8_cpu import cache, prefill, write


def test_a_pool_without_a_page():
    """(page 0 is what a page id beyond the pool is read as)"""
    none = {n: t[:0].contiguous() for n, t in cache().items()}
    for call in (write, prefill):
        with pytest.raises(KernelError, match="without a page"):
            call(**none)


@pytest.mark.parametrize("head_dim", [64, 128])
def test_a_launch_leaves_no_more_pieces_than_the_workspace_holds(head_dim):
    """On any device, whatever its number of SMs: shares by groups of warps, rows by pieces."""
    lib = kernels._kv8(head_dim)
    most, floats = lib.rl_kv8_most_pieces, lib.rl_kv8_part_floats
    most.restype, most.argtypes = ctypes.c_longlong, [ctypes.c_int] * 3
    floats.restype, floats.argtypes = ctypes.c_longlong, [ctypes.c_int]
    group = 4
    places = floats(group) // (2 * group * (head_dim + 4))
    warps = 12 if head_dim == 64 else 8
    for resident in (1, 2, 100, 147, 148, 149, 160, 192, 300, 1776, 1777, 5000):
        for groups in [n for n in range(1, warps + 1) if warps % n == 0]:
            assert 1 <= most(resident, groups, 0) <= places
            if resident <= 148:
                assert most(resident, groups, 0) == resident * groups
        for rows in (1, 3, 8, 64, 147, 148, 149, 1776, 1777, 2000):
            assert 0 <= most(resident, 1, rows) <= min(places, resident)
    assert most(148, 1, 8) == 144 and most(148, 1, 149) == 0
