"""Contexts for attention over the cache in 8 bits in which every 32 keys count: one of them, a needle, lies along the queries and has some
150 times the weight of the others, so a row's weight is spread evenly over its runs of 32 keys, and whatever is left out, taken twice or
read with another page's scale moves the result by more than the bound of ``tight`` (tests/test_kv8_ranges_gpu.py).  The scales differ
from page to page: of keys by an entry that the queries do not look at, of values by a factor."""

import math

import torch

import plain_kv8 as P


def blocks(x):
    """x [pages, heads, page, D] float32 as bytes and scales (plain_kv8.store of whole pages, all at once)."""
    mant, exp = torch.frexp(x.abs().amax((2, 3)))
    code = (exp - 9 + (mant > 0.875).int() + 127).clamp(1, 246)
    unit = torch.exp2(127.0 - code.double()).float()
    return (x * unit[:, :, None, None]).to(P.E4M3).view(torch.uint8), code.to(torch.uint8)


def needles(lengths, heads, kv_heads, dim, page, seed, directions=1, spread=1):
    """A cache (k, v, their scales), its block table, and queries [directions, sequences, heads, D] bfloat16: those of direction r
    look for the needles of every run of 32 keys number b with b % directions == r."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 1
    look = torch.randn(directions, kv_heads, dim, generator=g)
    look[..., 0] = 0.0
    look *= math.sqrt(dim) / look.norm(dim=-1, keepdim=True)
    table = torch.zeros(len(lengths), max(counts) + 1, dtype=torch.int32)
    order = torch.randperm(pages - 1, generator=g) + 1
    k, v = torch.zeros(pages, kv_heads, page, dim), torch.zeros(pages, kv_heads, page, dim)
    at = 0
    for s, c in enumerate(counts):
        mine = order[at:at + c]
        at += c
        table[s, :c] = mine.int()
        n = c * page
        keys = torch.randn(n, kv_heads, dim, generator=g) * 0.4
        runs = -(-lengths[s] // 32)
        place = torch.arange(runs) * 32 + torch.randint(0, 32, (runs,), generator=g)
        place[-1] = lengths[s] - 1 - int(torch.randint(0, lengths[s] - 32 * (runs - 1), (1,), generator=g))
        keys[place] = look[torch.arange(runs) % directions] * (5.0 / math.sqrt(dim))
        keys = keys.view(c, page, kv_heads, dim).transpose(1, 2)
        keys[..., 0] = 0.0
        keys[:, :, 0, 0] = torch.exp2(torch.randint(2, 9, (c, 1), generator=g).float())
        values = torch.randn(c, kv_heads, page, dim, generator=g) * torch.exp2(torch.randint(-spread, spread + 1, (c, 1, 1, 1), generator=g).float())
        k[mine], v[mine] = keys, values
    (kb, kc), (vb, vc) = blocks(k), blocks(v)
    kb[0], vb[0], kc[0], vc[0] = 0x7F, 0x7F, 255, 255          # what no sequence owns is not a number
    q = look[:, None].repeat_interleave(heads // kv_heads, 2).expand(-1, len(lengths), -1, -1)
    q = q * (1.0 + 0.1 * torch.rand(directions, len(lengths), heads, 1, generator=g)) + 0.05 * torch.randn(directions, len(lengths), heads, dim, generator=g)
    q[..., 0] = 0.0
    return [kb, vb, kc, vc], table, q.bfloat16()
