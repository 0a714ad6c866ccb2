"""Further refusals of the 8-bit cache's calls, without a GPU."""

import ctypes

import pytest
import torch

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


@pytest.mark.parametrize("head_dim,dtype,heads,impl", [(64, 0, 4, 2), (64, 0, 4, 4), (80, 1, 4, 3), (128, 1, 40, 2)])
def test_a_kernel_that_does_not_take_the_call_is_refused_first(head_dim, dtype, heads, impl):
    """Before the device is asked for anything, so before a token is stored (invalid argument, and not the error of a missing device)."""
    f = kernels._kv8(head_dim).rl_kv8_attn_decode
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_char_p]
    names = ("dtype q q_stride k v ks vs table blocks items nitems part counters out out_stride hq hkv page_size window scale cos sin "
             "max_pos store num_slots status max_ctx sum_ctx impl bad_page stream").split()
    values = dict.fromkeys(names, 0) | dict(dtype=dtype, nitems=1, hq=heads, hkv=2, page_size=16, scale=0.5, store=1, impl=impl)
    assert f(kernels._KV8_DECODE(*values.values())) == 1


def test_a_workspace_can_be_laid_out_anywhere():
    part, counters = kernels.kv8_decode_workspace(3, 4, 2, 64, torch.device("cpu"))
    assert part.numel() == kernels.kv8_part_floats(4, 2, 64) and counters.numel() == 6 and not counters.any()


@pytest.mark.parametrize("heads,kv_heads", [(4, 0), (0, 0), (0, 2), (4, -2), (4, 3), (2, 4)])
def test_heads_that_are_no_groups(heads, kv_heads):
    """Of every call that divides one number by the other."""
    cpu = torch.device("cpu")
    for call in (lambda: kernels.kv8_part_floats(heads, kv_heads, 64), lambda: kernels.kv8_decode_workspace(1, heads, kv_heads, 64, cpu),
                 lambda: kernels.kv8_decode_choice(torch.bfloat16, 1, heads, kv_heads, 64, 10, 10, 0, cpu),
                 lambda: write(num_heads=heads, num_kv_heads=kv_heads), lambda: prefill(num_heads=heads, num_kv_heads=kv_heads)):
        with pytest.raises(KernelError, match="no multiple"):
            call()
    if kv_heads < 1 or heads < kv_heads:
        assert kernels._kv8(64).rl_kv8_decode_choice(1, 1, heads, kv_heads, 10, ctypes.c_longlong(10)) == -1


def test_the_build_has_the_8_bit_cache_wherever_it_has_attention(monkeypatch):
    """(a head size that it leaves out is compiled within the first request)"""
    import __graft_entry__
    asked = {}
    monkeypatch.setattr(kernels, "build_all", lambda **kw: asked.update(kw))
    __graft_entry__.build()
    assert set(asked["head_dims"]) <= set(asked["kv8_dims"])


def test_native_calls_without_heads():
    """(what the Python checks refuse, asked of the library itself)"""
    lib = kernels._kv8(64)
    for f, fields in ((lib.rl_kv8_attn_decode, 31), (lib.rl_kv8_attn_prefill, 25)):
        f.restype, f.argtypes = ctypes.c_int, [ctypes.c_char_p]
        assert f(bytes(8 * fields)) == 1


@pytest.mark.parametrize("code,tc_code,said", [(4, 0, "a cache slot beyond the pool"), (8, 0, "a second run of tokens"), (0, 16, "a page id beyond the pool")])
def test_what_an_engine_says_of_the_bits(monkeypatch, code, tc_code, said):
    from types import SimpleNamespace
    from redline_b200.engine import runner
    word = torch.tensor([tc_code], dtype=torch.int32)
    monkeypatch.setattr(runner.kernels, "tc_status", lambda device: word)
    status = torch.tensor([code], dtype=torch.int32)
    me = SimpleNamespace(builder=SimpleNamespace(status=status), device=None)
    with pytest.raises(runner.EngineError, match=said):
        runner.ModelRunner.check_status(me)
    runner.ModelRunner.check_status(me)                  # (told once)
