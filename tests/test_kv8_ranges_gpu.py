"""Attention over the cache in 8 bits where numbers are not finite: what is not a number reaches the rows that see it and no others."""

import math

import pytest
import torch

import plain_kv8 as P
from redline_b200.ops import kernels
from test_kv8_gpu import DEV, DT, filled, near, on_gpu, tiles_of

pytestmark = pytest.mark.gpu


def prefill(q, gpu, table, segments, heads, kv_heads, dim, page, window, scale, impl):
    positions = torch.tensor([p for a, n in segments for p in range(a, a + n)], dtype=torch.int32, device=DEV)
    seq, tok, rows = tiles_of(segments)
    out = torch.full((len(q), heads * dim), 9.0, dtype=q.dtype, device=DEV)
    qg = q.to(DEV)
    kernels.kv8_attn_prefill(qg, qg.stride(0), *gpu, table.to(DEV), seq, tok, rows, positions, out, len(seq), heads, kv_heads, dim, page,
                             window, scale, impl=impl)
    assert kernels.tc_status(out.device).item() == 0
    return out


def same_where_finite(out, ref, v, dtype):
    """Not a number in the same places; elsewhere as near as ever."""
    ref = ref.to(out.device)
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(out), nan)
    near(torch.where(nan, torch.zeros_like(out), out), torch.where(nan, torch.zeros_like(ref), ref), v, dtype)


@pytest.mark.parametrize("heads,kv_heads,dim,page,window,dtype,impl", [
    (4, 2, 64, 16, 0, "bfloat16", 1), (4, 2, 64, 16, 0, "float32", 0), (3, 1, 128, 32, 0, "bfloat16", 1), (4, 2, 64, 64, 90, "float32", 0),
    (10, 2, 80, 16, 0, "bfloat16", 0), (2, 1, 16, 16, 25, "bfloat16", 0)])
def test_prompts_over_what_is_not_a_number(heads, kv_heads, dim, page, window, dtype, impl):
    """A key, an entry of a value and a page's scale in the middle of portions: the rows that see them, and only those."""
    segments = ((40, 200), (0, 70), (300, 150))
    lengths = [a + n for a, n in segments]
    cache, table = filled(lengths, heads, kv_heads, dim, page, seed=dim)

    def place(s, p):
        return int(table[s, p // page]), p % page

    b, r = place(0, 130)
    cache[1][b, 0, r, 3] = 0x7F                              # one entry of one value
    b, r = place(0, 200)
    cache[1][b, kv_heads - 1, r] = 0xFF                      # a whole value, not a number with a sign
    b, r = place(1, 33)
    cache[0][b, 0, r, 7] = 0x7F                              # a key
    b, _ = place(2, 400)
    cache[3][b, kv_heads - 1] = 255                          # a page's scale
    g = torch.Generator().manual_seed(3)
    q = torch.randn(sum(n for _, n in segments), heads * dim, generator=g).to(DT[dtype])
    scale = 1.0 / math.sqrt(dim)
    out = prefill(q, on_gpu(cache), table, segments, heads, kv_heads, dim, page, window, scale, impl)
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    v[cache[3] == 255] = math.nan
    row = 0
    for s, (a, n) in enumerate(segments):
        ref = P.attend(q[row:row + n].view(n, heads, dim), k, v, table[s], range(a, a + n), window, scale)
        assert torch.isnan(ref).any() and torch.isfinite(ref).any()
        same_where_finite(out[row:row + n].view(n, heads, dim), ref, v[table[s][:-(-lengths[s] // page)].long()], dtype)
        row += n


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [(4, 2, 64, 16, "bfloat16"), (16, 1, 128, 32, "bfloat16"), (4, 2, 64, 64, "float32"),
                                                           (10, 2, 80, 16, "bfloat16")])
@pytest.mark.parametrize("impl", [0, 1, 2, 3, 4])
def test_single_tokens_over_what_is_not_a_number(heads, kv_heads, dim, page, dtype, impl):
    if impl and (dtype == "float32" or dim == 80):
        pytest.skip("one way only")
    ctxs = (100, 200, 300, 64)
    cache, table = filled(ctxs, heads, kv_heads, dim, page, seed=2)
    cache[1][int(table[0, 50 // page]), 0, 50 % page, 3] = 0x7F
    cache[0][int(table[1, 199 // page]), kv_heads - 1, 199 % page, 9] = 0xFF
    cache[3][int(table[2, 0]), 0] = 255
    q = torch.randn(4, heads * dim, generator=torch.Generator().manual_seed(3)).to(DT[dtype])
    scale = 1.0 / math.sqrt(dim)
    items = torch.tensor([(i, i, c, 0) for i, c in enumerate(ctxs)], dtype=torch.int32, device=DEV)
    work = kernels.kv8_decode_workspace(4, heads, kv_heads, dim, torch.device(DEV))
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    v[cache[3] == 255] = math.nan
    for window in (0, 90):                                   # (with the window the third row no longer sees its page)
        qg, out = q.to(DEV), torch.empty(4, heads * dim, dtype=q.dtype, device=DEV)
        kernels.kv8_attn_decode(qg, qg.stride(0), *on_gpu(cache), table.to(DEV), items, work, out, 4, heads, kv_heads, dim, page, window,
                                scale, impl=impl)
        for s, n in enumerate(ctxs):
            ref = P.attend(q[s].view(1, heads, dim), k, v, table[s], [n - 1], window, scale)
            same_where_finite(out[s].view(1, heads, dim), ref, v[table[s][:-(-n // page)].long()], dtype)
