"""What the comparisons of test_kv8_long_gpu.py would notice, on the CPU: a run of 32 keys left out or taken twice, a page read with a scale
of another."""

import math

import pytest
import torch

import plain_kv8 as P
from kv8_needles import blocks, needles
from test_kv8_ranges_gpu import formula


def test_pages_as_the_restatement_stores_them():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 2, 16, 32, generator=g) * torch.exp2(torch.randint(-20, 20, (5, 2, 1, 1), generator=g).float())
    got = blocks(x)
    cache, scale = torch.zeros(5, 2, 16, 32, dtype=torch.uint8), torch.zeros(5, 2, dtype=torch.uint8)
    P.store(x.transpose(1, 2).reshape(80, 2, 32), range(80), cache, scale)
    assert torch.equal(got[0], cache) and torch.equal(got[1], scale)


@pytest.mark.parametrize("length,heads,kv_heads,dim,directions", [(2500, 4, 2, 64, 1), (9000, 4, 2, 64, 1), (5000, 3, 1, 128, 1), (70000, 4, 1, 64, 8),
                                                                  (7200, 4, 2, 64, 1)])
def test_the_bound_binds(length, heads, kv_heads, dim, directions):
    """Faults put into the formula's own result: each one is beyond the bound."""
    cache, table, queries = needles((length,), heads, kv_heads, dim, 16, 1, directions)
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    scale = 1.0 / math.sqrt(dim)
    runs = -(-length // 32)
    for b in (0, 1, 17, runs // 2, runs - 2, runs - 1):
        q = queries[b % directions, 0][None].float()
        ref, limit = formula(q, k, v, table[0], [length - 1], 0, scale, "bfloat16")
        page = table[0, 2 * b].long()                          # (a run of 32 keys begins a page)

        def differs(k, v, **change):
            wrong, _ = formula(q, k, v, table[0], [length - 1], 0, scale, "bfloat16", **change)
            return ((wrong - ref).abs() > limit).any(-1).all()      # in every head

        times = torch.ones(length, dtype=torch.float64)
        for n in (0.0, 2.0):                                   # left out; taken twice
            times[32 * b:32 * b + 32] = n
            assert differs(k, v, times=times)
        both = [p for p in table[0, 2 * b:2 * b + 2].long().tolist() if p]
        for t in (k, v):                                       # another page's scale
            was = t[both].clone()
            t[both] *= 2.0
            assert differs(k, v)
            t[both] = was
        assert page > 0
