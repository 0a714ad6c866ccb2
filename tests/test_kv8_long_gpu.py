"""Attention over long contexts in the cache of 8 bits: every run of 32 keys counts (kv8_needles.py), page scales differ from page to page,
and the bound is each number's own, so that a run left out, taken twice or read with another page's scale is noticed
(test_kv8_long_cpu.py).  Rows of many windows of 32 page ids, rows in pieces and shares that are put together again, groups of warps that take
rows one after another, prompts whose loaders ask for page ids many times over."""

import math

import pytest
import torch

import plain_kv8 as P
from kv8_needles import needles
from redline_b200.ops import kernels
from test_kv8_gpu import DEV, angles, on_gpu
from test_kv8_ranges_gpu import decode, prefill, tight

pytestmark = pytest.mark.gpu


MANY = tuple(2300 + 37 * i % 400 for i in range(40))
LONG = [  # heads, kv heads, head size, contexts, window, directions
    (32, 8, 64, MANY, 0, 1), (32, 8, 64, MANY, 1900, 1), (32, 8, 128, MANY[:24], 0, 1), (16, 8, 128, MANY[:24], 1777, 1),
    (16, 1, 64, (5000, 9000, 700, 2111), 0, 1), (16, 1, 128, (5000, 1234), 3000, 1),
    (4, 2, 64, (9000, 3, 70, 1, 400), 0, 1), (4, 2, 128, (5000,), 0, 1), (3, 1, 64, (70000,), 0, 8), (2, 1, 128, (40001, 20, 9), 0, 8),
]


@pytest.mark.parametrize("impl", [0, 2, 3, 4])
@pytest.mark.parametrize("heads,kv_heads,dim,ctxs,window,directions", LONG)
def test_single_tokens(heads, kv_heads, dim, ctxs, window, directions, impl):
    cache, table, queries = needles(ctxs, heads, kv_heads, dim, 16, 1, directions)
    gpu, scale = on_gpu(cache), 1.0 / math.sqrt(dim)
    k, v = (P.values(cache[i].to(DEV), cache[i + 2].to(DEV)) for i in (0, 1))
    for r in range(directions):
        q = queries[r]
        out = decode(q.reshape(len(ctxs), -1), gpu, table, ctxs, heads, kv_heads, dim, 16, window, scale, impl)
        for s, n in enumerate(ctxs):
            tight(out[s].view(1, heads, dim), q[s][None], k, v, table[s], [n - 1], window, scale, "bfloat16")


@pytest.mark.parametrize("impl", [0, 2, 3, 4])
@pytest.mark.parametrize("heads,kv_heads,dim,page,ctxs", [(32, 8, 64, 16, MANY), (16, 8, 128, 32, MANY[:24]), (4, 2, 64, 16, (9000, 1000, 33)),
                                                          (4, 1, 128, 16, (20001,)), (4, 2, 64, 64, (5000, 640, 641))])
def test_single_tokens_that_are_stored(heads, kv_heads, dim, page, ctxs, impl):
    """The token's own key and value among them, stored on the way."""
    cache, table, queries = needles(ctxs, heads, kv_heads, dim, page, 2)
    g = torch.Generator().manual_seed(1)
    n, scale = len(ctxs), 1.0 / math.sqrt(dim)
    cos, sin = angles(max(ctxs), dim)
    at = [c - 1 for c in ctxs]
    # q turned back by its angle, so that it looks the needles' way once it is rotated
    q = P.rotate(queries[0].float(), cos[at], -sin[at]).reshape(n, -1)
    x = torch.cat([q, torch.randn(n, 2 * kv_heads * dim, generator=g) * 2.0], 1).bfloat16()
    gpu = on_gpu(cache)
    items = torch.tensor([(i, i, c, 0) for i, c in enumerate(ctxs)], dtype=torch.int32, device=DEV)
    work = kernels.kv8_decode_workspace(n, heads, kv_heads, dim, torch.device(DEV))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    xg, out = x.to(DEV), torch.empty(n, heads * dim, dtype=x.dtype, device=DEV)
    kernels.kv8_attn_decode_rope(xg, xg.stride(0), *gpu, table.to(DEV), items, work, out, n, heads, kv_heads, dim, page, 0, scale,
                                 cos.to(DEV), sin.to(DEV), status, impl=impl)
    assert status.item() == 0 and (work[1] == 0).all()
    slots = [int(table[s, p // page]) * page + p % page for s, p in enumerate(at)]
    f = x.float()
    P.store(P.rotate(f[:, heads * dim:-kv_heads * dim].reshape(n, kv_heads, dim), cos[at], sin[at]), slots, cache[0], cache[2])
    P.store(f[:, -kv_heads * dim:].reshape(n, kv_heads, dim), slots, cache[1], cache[3])
    for got, want in zip(gpu, cache):
        assert torch.equal(got.view(torch.uint8).cpu(), want)
    k, v = (P.values(cache[i].to(DEV), cache[i + 2].to(DEV)) for i in (0, 1))
    q = P.rotate(f[:, :heads * dim].view(n, heads, dim), cos[at], sin[at])
    for s, c in enumerate(ctxs):
        tight(out[s].view(1, heads, dim), q[s:s + 1], k, v, table[s], [c - 1], 0, scale, "bfloat16", rounded_q=True)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("heads,kv_heads,dim,page,window,segments", [
    (4, 2, 64, 16, 0, ((7000, 200), (0, 130), (4100, 3))), (4, 2, 64, 16, 5000, ((7000, 200),)), (3, 1, 128, 16, 0, ((5000, 140), (2, 129))),
    (2, 2, 64, 32, 0, ((6900, 300),)), (2, 1, 128, 64, 2500, ((5000, 260),))])
def test_prompts(heads, kv_heads, dim, page, window, segments, impl):
    lengths = [a + n for a, n in segments]
    cache, table, queries = needles(lengths, heads, kv_heads, dim, page, 3)
    g = torch.Generator().manual_seed(2)
    q = torch.cat([queries[0, s][None].float() * (1.0 + 0.1 * torch.rand(n, heads, 1, generator=g)) for s, (_, n) in enumerate(segments)]).bfloat16()
    scale = 1.0 / math.sqrt(dim)
    out = prefill(q.view(len(q), -1), on_gpu(cache), table, segments, heads, kv_heads, dim, page, window, scale, impl)
    k, v = (P.values(cache[i].to(DEV), cache[i + 2].to(DEV)) for i in (0, 1))
    row = 0
    for s, (a, n) in enumerate(segments):
        tight(out[row:row + n].view(n, heads, dim), q[row:row + n], k, v, table[s], range(a, a + n), window, scale, "bfloat16")
        row += n
