"""The cache in 8 bits: its write, single-token and prompt attention, against a restatement with elementary operations
(plain_kv8.py) and attention in float64.

The write is compared bit for bit.  Attention, with E the largest magnitude among a kv head's values:
  float32   |error| <= 2e-5 E: sums and exponentials in float32 (2^-22 each, a few hundred keys in chains)
  bfloat16  |error| <= 2^-8 |result| + (2^-8 + 2e-5) E: the result's one rounding, and the softmax weights' (bfloat16 at most;
            their roundings weigh the values, so their sum is at most half a step of E)"""

import math
import os
import subprocess
import sys

import pytest
import torch

import plain_kv8 as P
from redline_b200.ops import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def near(got, ref, v, dtype):
    ref = ref.to(got.device)
    most = v[torch.isfinite(v)].abs().max().item()
    err = (got.double() - ref).abs()
    limit = 2e-5 * most if dtype == "float32" else 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2e-5) * most
    assert torch.isfinite(got).all()
    assert (err <= limit).all(), f"error {err.max().item():.3e}, {(err / torch.as_tensor(limit)).max().item():.2f} of the limit"


def angles(n, dim):
    a = torch.arange(n, dtype=torch.float64)[:, None] * (10000.0 ** (-2.0 * torch.arange(dim // 2) / dim))
    return torch.cos(a).float(), torch.sin(a).float()


def empty_cache(pages, heads, page, dim, seed=0):
    """Bytes that an earlier owner left, and scales likewise."""
    g = torch.Generator().manual_seed(seed)
    cache = [(torch.randint(0, 127, (pages, heads, page, dim), generator=g)
              + 128 * torch.randint(0, 2, (pages, heads, page, dim), generator=g)).to(torch.uint8) for _ in range(2)]
    scale = [torch.randint(0, 255, (pages, heads), generator=g).to(torch.uint8) for _ in range(2)]
    return cache + scale


def on_gpu(cache):
    k, v, ks, vs = (t.to(DEV) for t in cache)
    return k.view(P.E4M3), v.view(P.E4M3), ks.view(P.E8M0), vs.view(P.E8M0)


def check_write(x, positions, slots, cos, sin, cache, heads, kv_heads, dim, page, expect_status=0, q_out=None, tokens=None):
    """One call on the GPU and the restatement on the CPU: the same bytes everywhere, the same q."""
    T = len(positions) if tokens is None else tokens
    gpu = on_gpu(cache)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    xg = x.to(DEV)
    out = torch.full((x.shape[0], heads * dim), 7.0, dtype=x.dtype, device=DEV) if q_out is None else q_out(xg)
    kernels.kv8_write(xg, torch.tensor(positions, dtype=torch.int32, device=DEV),
                      None if slots is None else torch.tensor(slots, dtype=torch.int32, device=DEV),
                      None if cos is None else cos.to(DEV), None if sin is None else sin.to(DEV), *gpu, out, heads, kv_heads, dim,
                      page, status, tokens=tokens)
    q, k, v = x.float().split([heads * dim, kv_heads * dim, kv_heads * dim], -1)
    q, k, v = q.view(-1, heads, dim)[:T], k.view(-1, kv_heads, dim)[:T], v.view(-1, kv_heads, dim)[:T]
    if cos is not None:
        at = torch.tensor(positions[:T]).long()
        q, k = P.rotate(q, cos[at], sin[at]), P.rotate(k, cos[at], sin[at])
    if slots is not None:
        P.store(k, slots[:T], cache[0], cache[2])
        P.store(v, slots[:T], cache[1], cache[3])
    for name, got, want in zip(("k", "v", "k scales", "v scales"), gpu, cache):
        same = got.view(torch.uint8).cpu() == want
        assert same.all(), f"{name}: {(~same).sum().item()} bytes differ, the first at {(~same).nonzero()[0].tolist()}"
    assert torch.equal(out[:T].cpu(), q.reshape(T, -1).to(x.dtype))
    assert status.item() == expect_status
    return out


def rows_of(segments, table, page):
    """positions and slots of segments (start, new tokens), sequence by sequence."""
    positions, slots = [], []
    for s, (start, n) in enumerate(segments):
        for p in range(start, start + n):
            positions.append(p)
            slots.append(int(table[s][p // page]) * page + p % page)
    return positions, slots


LAYOUTS = [(4, 2, 16), (3, 1, 64), (10, 2, 80), (4, 2, 128), (2, 2, 256)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
def test_write(heads, kv_heads, dim, page, dtype):
    """Whole prompts, portions that begin within a page, single tokens; then the next steps on the same pages."""
    g = torch.Generator().manual_seed(dim + page)
    pages = 24
    cache = empty_cache(pages, kv_heads, page, dim, seed=1)
    order = torch.randperm(pages - 1, generator=g) + 1
    table = order[:20].view(5, 4)
    cos, sin = angles(4 * page, dim)
    at = [0, 0, 0, 0, 0]
    for step, news in enumerate([(page + 5, 1, 2 * page, 3, 7), (1, 1, 1, 1, 1), (page - 5, 4, 17, 1, page), (1, 2, 1, 30, 1)]):
        segments = list(zip(at, news))
        positions, slots = rows_of(segments, table, page)
        x = torch.randn(len(positions), (heads + 2 * kv_heads) * dim, generator=g)
        x *= torch.exp2(torch.randint(-6, 7, (len(positions), 1), generator=g).float())      # (scales that rise now and then)
        check_write(x.to(DT[dtype]), positions, slots, cos, sin, cache, heads, kv_heads, dim, page)
        at = [a + n for a, n in segments]


def test_write_of_blocks_that_need_care():
    """Zeros, numbers below the smallest scale, numbers beyond the largest, infinities and not-a-numbers, borders."""
    heads, kv_heads, dim, page = 2, 1, 64, 16
    g = torch.Generator().manual_seed(3)
    table = [[1], [2], [3], [4], [5], [6], [7], [8]]
    blocks = [torch.zeros(16, dim), torch.randn(16, dim, generator=g) * 2.0 ** -130, torch.randn(16, dim, generator=g) * 1e38,
              torch.full((16, dim), math.inf), torch.randn(16, dim, generator=g), torch.full((16, dim), 448.0),
              torch.full((16, dim), 449.0), torch.full((16, dim), 2.0 ** -9)]
    blocks[4][3, 5], blocks[4][0, 0], blocks[4][7, 1] = math.inf, math.nan, -math.inf
    blocks[2].clamp_(-3.3e38, 3.3e38)
    x = torch.cat([torch.randn(128, heads * dim, generator=g), torch.cat(blocks), torch.cat(blocks[::-1])], 1)
    positions, slots = rows_of([(0, 16)] * 8, table, page)
    check_write(x, positions, slots, None, None, empty_cache(9, kv_heads, page, dim, 2), heads, kv_heads, dim, page)
    # behind a page's first tokens: what is there is rescaled, or the scale stays
    cache = empty_cache(9, kv_heads, page, dim, 2)
    for t in table:                                     # (finite bytes before the new ones, scales of all sizes)
        cache[0][t[0]] = torch.randint(0, 127, (kv_heads, page, dim), generator=g).to(torch.uint8)
        cache[1][t[0]] = torch.randint(128, 255, (kv_heads, page, dim), generator=g).to(torch.uint8)
    cache[2][1:], cache[3][1:] = torch.arange(8)[:, None].to(torch.uint8) * 32, torch.arange(8)[:, None].to(torch.uint8) * 20 + 90
    positions, slots = rows_of([(5, 3)] * 8, table, page)
    keep = torch.cat([torch.arange(16 * s, 16 * s + 3) for s in range(8)])
    check_write(x[keep].contiguous(), positions, slots, None, None, cache, heads, kv_heads, dim, page)


def test_write_of_chosen_tokens():
    """No slot, a slot beyond the pool (told), tokens behind the call's, a page named by two runs (the first stays, told), page 0."""
    heads, kv_heads, dim, page = 4, 2, 16, 16
    g = torch.Generator().manual_seed(4)
    cos, sin = angles(64, dim)
    n = 12
    x = torch.randn(n, (heads + 2 * kv_heads) * dim, generator=g).bfloat16()
    positions = list(range(n))

    def run(slots, status, **kw):
        check_write(x, positions, slots, cos, sin, empty_cache(4, kv_heads, page, dim, 5), heads, kv_heads, dim, page, status, **kw)

    run([16, 17, -1, -1, 35, 36, 37, -1, 48, 49, -1, 50], 8)      # (50: a second run of page 3)
    run([16, 17, 18, 4 * page, 4 * page + 1, 33, 34, 2 ** 30, 48, 49, 50, 51], 4)
    run([16, 16, 16, 33, 33, 34, 48, 49, 50, 51, 52, 53], 8)
    run([0, 0, 0, 0, 1, 2, 3, 40, 41, 42, 43, 44], 0)
    run([16, 17, 18, 33, 34, 35, 36, 37, 48, 49, 50, 51], 0, tokens=7)
    run([-1] * n, 0)
    run(None, 0)


def test_write_out_of_place_in_place_and_strided():
    heads, kv_heads, dim, page, n = 4, 2, 64, 16, 9
    g = torch.Generator().manual_seed(6)
    cos, sin = angles(32, dim)
    wide = torch.randn(n, (heads + 2 * kv_heads) * dim + 24, generator=g).bfloat16()
    positions, slots = rows_of([(3, 5), (0, 4)], [[2], [1]], page)
    x = wide[:, 8:8 + (heads + 2 * kv_heads) * dim]
    cache = empty_cache(3, kv_heads, page, dim)
    check_write(x, positions, slots, cos, sin, cache, heads, kv_heads, dim, page)
    # in place: q's columns of qkv itself, k and v as they were
    cache = empty_cache(3, kv_heads, page, dim)
    seen = []
    check_write(x, positions, slots, cos, sin, cache, heads, kv_heads, dim, page,
                q_out=lambda xg: (seen.append(xg), xg[:, :heads * dim])[1])
    assert torch.equal(seen[0][:, heads * dim:].cpu(), x[:, heads * dim:])
    # no q wanted; a position beyond the tables is told
    gpu, status = on_gpu(empty_cache(3, kv_heads, page, dim)), torch.zeros(1, dtype=torch.int32, device=DEV)
    late = torch.tensor([3, 4, 5, 6, 99, 0, 1, 2, 3], dtype=torch.int32, device=DEV)
    xg = x.to(DEV)
    kernels.kv8_write(xg, late, torch.tensor(slots, dtype=torch.int32, device=DEV), cos.to(DEV), sin.to(DEV), *gpu, None, heads,
                      kv_heads, dim, page, status)
    assert status.item() == 2


def filled(lengths, heads, kv_heads, dim, page, seed, spread=0.3, poison=True):
    """A cache with sequences of these lengths on shuffled pages, and its block table; what no sequence owns is not a number."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-n // page) for n in lengths]
    pages = sum(blocks) + 2
    cache = empty_cache(pages, kv_heads, page, dim, seed)
    if poison:
        cache[0].fill_(0x7F)
        cache[1].fill_(0xFF)
        cache[2].fill_(255)
        cache[3].fill_(255)
    order = (torch.randperm(pages - 1, generator=g) + 1).tolist()
    table = torch.zeros(len(lengths), max(blocks + [1]) + 1, dtype=torch.int32)
    x = []
    for s, (n, b) in enumerate(zip(lengths, blocks)):
        mine, order = order[:b], order[b:]
        table[s, :b] = torch.tensor(mine, dtype=torch.int32)
        for name in (0, 1):
            data = torch.randn(n, kv_heads, dim, generator=g)
            data *= torch.exp2(torch.randn(n, 1, 1, generator=g) * spread)
            slot = [mine[p // page] * page + p % page for p in range(n)]
            P.store(data, slot, cache[name], cache[name + 2])
            x.append(data)
    return cache, table


def decode(q, cache, table, ctxs, heads, kv_heads, dim, page, window, scale, order=None, out=None, **kw):
    n = len(ctxs)
    items = torch.zeros(n, 4, dtype=torch.int32)
    items[:, 0] = torch.arange(n) if order is None else torch.tensor(order)
    items[:, 1] = torch.arange(n)
    items[:, 2] = torch.tensor(ctxs)
    work = kernels.kv8_decode_workspace(n, heads, kv_heads, dim, torch.device(DEV))
    out = torch.full((q.shape[0], heads * dim), 9.0, dtype=q.dtype, device=DEV) if out is None else out
    kernels.kv8_attn_decode(q, q.stride(0), *cache, table.to(DEV), items.to(DEV), work, out, n, heads, kv_heads, dim, page, window,
                            scale, **kw)
    assert (work[1] == 0).all()
    return out


DECODE = [  # heads, kv heads, head size, page, window, contexts
    (4, 2, 64, 16, 0, (1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 130)),
    (32, 8, 64, 16, 0, (513, 40)),
    (8, 8, 64, 32, 0, (300, 1, 77)),
    (16, 1, 128, 16, 0, (257, 1000, 5)),
    (24, 2, 64, 64, 0, (200, 129)),
    (40, 2, 64, 16, 0, (90, 33)),
    (3, 1, 128, 64, 0, (1, 64, 65, 700)),
    (12, 4, 128, 32, 50, (1, 49, 50, 51, 400)),
    (4, 2, 64, 16, 33, (16, 33, 34, 47, 48, 49, 64, 65, 66, 200)),
    (10, 2, 80, 16, 0, (1, 100, 333)),
    (4, 2, 16, 16, 7, (1, 8, 90)),
    (6, 2, 96, 32, 0, (64, 511)),
    (8, 1, 256, 16, 0, (2, 65, 300)),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,kv_heads,dim,page,window,ctxs", DECODE)
@pytest.mark.parametrize("impl", [0, 1, 2, 3, 4])
def test_decode(heads, kv_heads, dim, page, window, ctxs, dtype, impl):
    if impl >= 2 and (dtype == "float32" or dim not in (64, 128) or heads > 16 * kv_heads):
        with pytest.raises(kernels.KernelError):
            cache, table = filled((3,), heads, kv_heads, dim, page, seed=1)
            decode(torch.zeros(1, heads * dim, dtype=DT[dtype], device=DEV), on_gpu(cache), table, (3,), heads, kv_heads, dim, page, 0,
                   1.0, impl=impl)
        return
    cache, table = filled(ctxs, heads, kv_heads, dim, page, seed=dim + len(ctxs))
    g = torch.Generator().manual_seed(9)
    q = torch.randn(len(ctxs), heads * dim, generator=g).to(DT[dtype])
    scale = 1.0 / math.sqrt(dim)
    out = decode(q.to(DEV), on_gpu(cache), table, ctxs, heads, kv_heads, dim, page, window, scale, impl=impl)
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    for s, n in enumerate(ctxs):
        ref = P.attend(q[s].view(1, heads, dim), k, v, table[s], [n - 1], window, scale)
        mine = v[table[s][:-(-n // page)].long()]
        near(out[s].view(1, heads, dim), ref, mine, dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_of_many_and_of_very_different_lengths(dim, dtype):
    """More rows than an SM each; one long row among short ones: rows that are cut and put together again, twice the same bits."""
    heads, kv_heads, page = 4, 2, 16
    g = torch.Generator().manual_seed(dim)
    for ctxs in (tuple(int(x) for x in torch.randint(1, 150, (150,), generator=g)), (9000, 3, 70, 1, 400), (5000,), (1,) * 300):
        cache, table = filled(ctxs, heads, kv_heads, dim, page, seed=2)
        q = torch.randn(len(ctxs), heads * dim, generator=g).to(DT[dtype])
        scale = 1.0 / math.sqrt(dim)
        gpu, qg = on_gpu(cache), q.to(DEV)
        out = decode(qg, gpu, table, ctxs, heads, kv_heads, dim, page, 0, scale)
        k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
        for s in list(range(len(ctxs)))[:12]:
            ref = P.attend(q[s].view(1, heads, dim), k, v, table[s], [ctxs[s] - 1], 0, scale)
            near(out[s].view(1, heads, dim), ref, v[table[s][:-(-ctxs[s] // page)].long()], dtype)
        again = decode(qg, gpu, table, ctxs, heads, kv_heads, dim, page, 0, scale)
        assert torch.equal(out, again)
        for kw in (dict(max_ctx=max(ctxs), sum_ctx=sum(ctxs)), dict(impl=1)) + ((dict(impl=2), dict(impl=3), dict(impl=4)) if dtype == "bfloat16" else ()):
            told = decode(qg, gpu, table, ctxs, heads, kv_heads, dim, page, 0, scale, **kw)
            for s in range(len(ctxs)):      # (another way to share the work out: other last bits)
                mine = v[table[s][:-(-ctxs[s] // page)].long()]
                near(told[s], out[s].double(), mine, dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_decode_of_scales_far_apart(dtype):
    """Blocks of values 2^20 apart and blocks of zeros; keys that make one far key take all the weight."""
    heads, kv_heads, dim, page, n = 4, 1, 64, 16, 200
    cache, table = filled((n,), heads, kv_heads, dim, page, seed=5)
    for b, p in enumerate(table[0].tolist()):
        if p:
            cache[3][p] = 127 + (-20 if b % 3 == 0 else 0)
            if b % 3 == 1:
                cache[1][p] = 0
                cache[3][p] = 1
    g = torch.Generator().manual_seed(1)
    scale = 1.0 / math.sqrt(dim)
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    for q in (torch.randn(1, heads * dim, generator=g), 12.0 * k[int(table[0, 3]), 0, 5].float().repeat(heads).view(1, -1),
              torch.randn(1, heads * dim, generator=g) * 2.0 ** 60, torch.zeros(1, heads * dim)):
        q = q.to(DT[dtype])
        out = decode(q.to(DEV), on_gpu(cache), table, (n,), heads, kv_heads, dim, page, 0, scale)
        ref = P.attend(q.view(1, heads, dim), k, v, table[0], [n - 1], 0, scale)
        near(out.view(1, heads, dim), ref, v[table[0][:-(-n // page)].long()], dtype)


@pytest.mark.parametrize("dim", [64, 80])
def test_decode_leaves_rows_without_keys(dim):
    """An item of context 0; rows of out that no item names; items in another order than their tokens; wide rows."""
    heads, kv_heads, page = 4, 2, 16
    ctxs = (40, 1, 70)
    cache, table = filled(ctxs, heads, kv_heads, dim, page, seed=4)
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(6, heads * dim + 16, generator=g).bfloat16()
    q = wide.to(DEV)[:, 8:8 + heads * dim]
    big = torch.full((6, heads * dim + 32), 5.0, dtype=torch.bfloat16, device=DEV)
    scale = 0.2
    out = decode(q, on_gpu(cache), table, (40, 0, 70), heads, kv_heads, dim, page, 0, scale, order=[4, 2, 0], out=big[:, 16:16 + heads * dim])
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    for s, row in ((0, 4), (2, 0)):
        ref = P.attend(wide[row, 8:8 + heads * dim].view(1, heads, dim), k, v, table[s], [ctxs[s] - 1], 0, scale)
        near(out[row].view(1, heads, dim), ref, v[table[s][:-(-ctxs[s] // page)].long()], "bfloat16")
    untouched = big.clone()
    untouched[4, 16:16 + heads * dim] = untouched[0, 16:16 + heads * dim] = 5.0
    assert (untouched == 5.0).all()
    none = decode(q, on_gpu(cache), table, (0, 0, 0), heads, kv_heads, dim, page, 0, scale)
    assert (none == 9.0).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,kv_heads,dim,page,window", [(4, 2, 64, 16, 0), (32, 8, 64, 32, 0), (4, 1, 128, 64, 40), (10, 2, 80, 16, 0),
                                                            (12, 1, 128, 16, 0), (20, 2, 64, 16, 35), (8, 1, 128, 32, 0)])
@pytest.mark.parametrize("impl", [0, 2, 3, 4])
def test_decode_with_the_tokens_own_keys(heads, kv_heads, dim, page, window, dtype, impl):
    """Rows [q | k | v] as the projection leaves them: stored and attended, against the write and the attention one after another."""
    if impl and (dtype == "float32" or dim == 80):
        pytest.skip("one way only")
    ctxs = (1, 2, 16, 17, 32, 64, 65, 200, 333)
    cache, table = filled([max(n - 1, 1) for n in ctxs], heads, kv_heads, dim, page, seed=8, poison=False)
    spare = int(table.max()) + 1
    g = torch.Generator().manual_seed(3)
    pages = cache[0].shape[0] + len(ctxs)
    grown = empty_cache(pages, kv_heads, page, dim, 1)
    for old, new in zip(cache, grown):
        new[:old.shape[0]] = old
    cache = grown
    nxt = pages - len(ctxs)
    for s, n in enumerate(ctxs):                      # a page for a token that begins one
        if (n - 1) % page == 0:
            table[s, (n - 1) // page] = nxt
            nxt += 1
    assert spare <= pages
    x = torch.randn(len(ctxs), (heads + 2 * kv_heads) * dim, generator=g)
    x *= torch.exp2(torch.randint(-3, 4, (len(ctxs), 1), generator=g).float())
    x = x.to(DT[dtype])
    cos, sin = angles(400, dim)
    scale = 1.0 / math.sqrt(dim)
    gpu = on_gpu(cache)
    items = torch.tensor([(i, i, n, 0) for i, n in enumerate(ctxs)], dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    work = kernels.kv8_decode_workspace(len(ctxs), heads, kv_heads, dim, torch.device(DEV))
    for _ in range(2):                                # (a step that is run again gives the same)
        out = torch.empty(len(ctxs), heads * dim, dtype=x.dtype, device=DEV)
        xg = x.to(DEV)
        kernels.kv8_attn_decode_rope(xg, xg.stride(0), *gpu, table.to(DEV), items, work, out, len(ctxs), heads, kv_heads, dim, page,
                                     window, scale, cos.to(DEV), sin.to(DEV), status, max_ctx=max(ctxs), sum_ctx=sum(ctxs), impl=impl)
        assert torch.equal(xg.cpu(), x) and status.item() == 0
        positions = [n - 1 for n in ctxs]
        slots = [int(table[s, p // page]) * page + p % page for s, p in enumerate(positions)]
        check_write(x, positions, slots, cos, sin, cache, heads, kv_heads, dim, page)
        q = P.rotate(x.float()[:, :heads * dim].view(-1, heads, dim), cos[positions], sin[positions])     # (not rounded on its way)
        for got, want in zip(gpu, cache):
            assert torch.equal(got.view(torch.uint8).cpu(), want)
        k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
        for s, n in enumerate(ctxs):
            ref = P.attend(q[s].view(1, heads, dim), k, v, table[s], [n - 1], window, scale)
            near(out[s].view(1, heads, dim), ref, v[table[s][:-(-n // page)].long()], dtype)
    items[3, 2] = 500                                 # a position beyond the tables is told, and nothing beyond them is read
    kernels.kv8_attn_decode_rope(xg, xg.stride(0), *gpu, torch.zeros(len(ctxs), 500 // page + 1, dtype=torch.int32, device=DEV), items,
                                 work, out, len(ctxs), heads, kv_heads, dim, page, window, scale, cos.to(DEV), sin.to(DEV), status)
    assert status.item() & 2


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [(4, 2, 64, 16, "bfloat16"), (4, 2, 64, 64, "bfloat16"), (4, 2, 64, 16, "float32"),
                                                           (10, 2, 80, 32, "bfloat16"), (4, 1, 128, 64, "bfloat16")])
def test_decode_of_items_in_another_order(heads, kv_heads, dim, page, dtype):
    """Items name their rows: in another order than the rows, and only some of them, they store and attend the same."""
    ctxs = (1, 17, 33, 64, 130)
    cache, table = filled([max(n - 1, 1) for n in ctxs], heads, kv_heads, dim, page, seed=9, poison=False)
    pages = cache[0].shape[0] + len(ctxs)
    grown = empty_cache(pages, kv_heads, page, dim, 1)
    for old, new in zip(cache, grown):
        new[:old.shape[0]] = old
    for s, n in enumerate(ctxs):
        if (n - 1) % page == 0:
            table[s, (n - 1) // page] = pages - 1 - s
    g = torch.Generator().manual_seed(5)
    x = torch.randn(len(ctxs) + 2, (heads + 2 * kv_heads) * dim, generator=g).to(DT[dtype]).to(DEV)
    cos, sin = (t.to(DEV) for t in angles(140, dim))
    work = kernels.kv8_decode_workspace(len(ctxs), heads, kv_heads, dim, torch.device(DEV))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    results = []
    row_of = (6, 2, 0, 5, 3)
    for order in ((0, 1, 2, 3, 4), (3, 0, 4, 2, 1)):
        gpu = on_gpu(grown)
        out = torch.full((len(x), heads * dim), 9.0, dtype=x.dtype, device=DEV)
        items = torch.tensor([(row_of[s], s, ctxs[s], 0) for s in order], dtype=torch.int32, device=DEV)
        kernels.kv8_attn_decode_rope(x, x.stride(0), *gpu, table.to(DEV), items, work, out, len(order), heads, kv_heads, dim, page, 0,
                                     1.0 / math.sqrt(dim), cos, sin, status, max_ctx=max(ctxs), sum_ctx=sum(ctxs))
        results.append((out, *(t.view(torch.uint8).cpu() for t in gpu)))
    assert status.item() == 0
    positions = [n - 1 for n in ctxs]
    slots = [int(table[s, p // page]) * page + p % page for s, p in enumerate(positions)]
    k, v = (x.cpu().float()[list(row_of)][:, (heads + i * kv_heads) * dim:][:, :kv_heads * dim].reshape(-1, kv_heads, dim) for i in (0, 1))
    P.store(P.rotate(k, cos.cpu()[positions], sin.cpu()[positions]), slots, grown[0], grown[2])
    P.store(v, slots, grown[1], grown[3])
    for out, *stored in results:
        for got, want in zip(stored, grown):
            assert torch.equal(got, want)
        assert (out[[1, 4]] == 9.0).all()
        keys, vals = P.values(grown[0], grown[2]), P.values(grown[1], grown[3])
        for s, n in enumerate(ctxs):
            q = P.rotate(x.cpu().float()[row_of[s], :heads * dim].view(1, heads, dim), cos.cpu()[n - 1:n], sin.cpu()[n - 1:n])
            ref = P.attend(q, keys, vals, table[s], [n - 1], 0, 1.0 / math.sqrt(dim))
            near(out[row_of[s]].view(1, heads, dim), ref, vals[table[s][:-(-n // page)].long()], dtype)


PROMPT = [  # heads, kv heads, head size, page, window, (cached, new) of every sequence
    (4, 2, 64, 16, 0, ((0, 2), (0, 33), (5, 128), (100, 129))),
    (32, 8, 64, 16, 0, ((70, 200),)),
    (3, 1, 64, 32, 0, ((0, 64), (63, 65))),
    (3, 1, 128, 16, 0, ((17, 140), (0, 5))),
    (8, 2, 128, 64, 0, ((0, 300),)),
    (4, 2, 64, 16, 20, ((0, 150), (300, 40))),
    (4, 4, 128, 32, 130, ((200, 260),)),
    (10, 2, 80, 16, 0, ((0, 70), (33, 66))),
    (6, 2, 96, 32, 9, ((40, 70),)),
    (4, 2, 16, 16, 0, ((3, 100),)),
    (2, 1, 256, 16, 0, ((20, 90),)),
]


def tiles_of(segments):
    tiles, row = [], 0
    for s, (_, n) in enumerate(segments):
        tiles += [(s, row + i, min(128, n - i)) for i in range(0, n, 128)]
        row += n
    return [torch.tensor(t, dtype=torch.int32, device=DEV) for t in zip(*tiles)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,kv_heads,dim,page,window,segments", PROMPT)
@pytest.mark.parametrize("impl", [0, 1])
def test_prefill(heads, kv_heads, dim, page, window, segments, dtype, impl):
    lengths = [a + n for a, n in segments]
    cache, table = filled(lengths, heads, kv_heads, dim, page, seed=dim)
    g = torch.Generator().manual_seed(7)
    T = sum(n for _, n in segments)
    q = torch.randn(T + 3, heads * dim, generator=g).to(DT[dtype])
    positions = torch.tensor([p for a, n in segments for p in range(a, a + n)] + [0, 0, 0], dtype=torch.int32, device=DEV)
    seq, tok, rows = tiles_of(segments)
    out = torch.full((T + 3, heads * dim), 9.0, dtype=q.dtype, device=DEV)
    scale = 1.0 / math.sqrt(dim)
    qg = q.to(DEV)
    kernels.kv8_attn_prefill(qg, qg.stride(0), *on_gpu(cache), table.to(DEV), seq, tok, rows, positions, out, len(seq), heads,
                             kv_heads, dim, page, window, scale, impl=impl)
    assert kernels.tc_status(out.device).item() == 0
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    row = 0
    for s, (a, n) in enumerate(segments):
        ref = P.attend(q[row:row + n].view(n, heads, dim), k, v, table[s], range(a, a + n), window, scale)
        near(out[row:row + n].view(n, heads, dim), ref, v[table[s][:-(-lengths[s] // page)].long()], dtype)
        row += n
    assert (out[T:] == 9.0).all()                     # rows behind the last sequence stay as they were


@pytest.mark.parametrize("heads,kv_heads,dim,page,window,segments", [
    (32, 8, 64, 16, 0, ((900, 1500), (0, 700), (10, 1))), (32, 8, 128, 16, 0, ((700, 1400), (0, 900))),
    (24, 8, 128, 64, 300, ((0, 1300), (2000, 1000))), (8, 8, 64, 32, 0, ((0, 2600), (300, 1500)))])
def test_prefill_of_more_items_than_sms(heads, kv_heads, dim, page, window, segments):
    """Several items to a CTA, of one key tile and of many, groups of one, three and four heads; some rows of every tile looked at."""
    lengths = [a + n for a, n in segments]
    cache, table = filled(lengths, heads, kv_heads, dim, page, seed=1)
    g = torch.Generator().manual_seed(8)
    T = sum(n for _, n in segments)
    q = torch.randn(T, heads * dim, generator=g).bfloat16()
    positions = torch.tensor([p for a, n in segments for p in range(a, a + n)], dtype=torch.int32, device=DEV)
    seq, tok, rows = tiles_of(segments)
    out = torch.full((T, heads * dim), 9.0, dtype=q.dtype, device=DEV)
    scale = 1.0 / math.sqrt(dim)
    qg = q.to(DEV)
    kernels.kv8_attn_prefill(qg, qg.stride(0), *on_gpu(cache), table.to(DEV), seq, tok, rows, positions, out, len(seq), heads,
                             kv_heads, dim, page, window, scale)
    assert kernels.tc_status(out.device).item() == 0
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    row = 0
    for s, (a, n) in enumerate(segments):
        for i in sorted({*range(0, n, 128), *range(77, n, 128), n - 1}):
            ref = P.attend(q[row + i:row + i + 1].view(1, heads, dim), k, v, table[s], [a + i], window, scale)
            near(out[row + i:row + i + 1].view(1, heads, dim), ref, v[table[s][:-(-lengths[s] // page)].long()], "bfloat16")
        row += n


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 64, 16), (4, 1, 128, 32), (10, 2, 80, 64)])
def test_a_run_of_steps(heads, kv_heads, dim, page, dtype):
    """Two sequences as an engine drives them: prompts in portions beside single tokens of the other, then tokens together, captured
    into a graph and replayed; every row against attention in float64 over what is stored by then."""
    g = torch.Generator().manual_seed(11)
    pages = 40
    cache = empty_cache(pages, kv_heads, page, dim, 3)
    gpu = on_gpu(cache)
    table = (torch.randperm(pages - 1, generator=g) + 1)[:38].view(2, 19).int()
    cos, sin = angles(300, dim)
    cg, sg, tg = cos.to(DEV), sin.to(DEV), table.to(DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    work = kernels.kv8_decode_workspace(2, heads, kv_heads, dim, torch.device(DEV))
    scale = 1.0 / math.sqrt(dim)
    width = (heads + 2 * kv_heads) * dim
    at = [0, 0]

    def compare(out, q, segments):
        k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
        row = 0
        for s, (a, n) in segments:
            ref = P.attend(q[row:row + n].cpu().view(n, heads, dim), k, v, table[s], range(a, a + n), 0, scale)
            near(out[row:row + n].view(n, heads, dim), ref, v[table[s][:-(-(a + n) // page)].long()], dtype)
            row += n

    for news in ((130, 0), (1, 45), (40, 1), (1, 20)):
        segments = [(s, (at[s], n)) for s, n in enumerate(news) if n]
        positions, slots = [], []
        for s, (a, n) in segments:
            p, t = rows_of([(a, n)], table[s:s + 1], page)
            positions += p
            slots += t
        x = torch.randn(len(positions), width, generator=g).to(DT[dtype])
        P.store(P.rotate(x.float()[:, heads * dim:-kv_heads * dim].view(-1, kv_heads, dim), cos[positions], sin[positions]), slots,
                cache[0], cache[2])
        P.store(x.float()[:, -kv_heads * dim:].reshape(-1, kv_heads, dim), slots, cache[1], cache[3])
        xg = x.to(DEV)
        pos = torch.tensor(positions, dtype=torch.int32, device=DEV)
        q = torch.empty(len(positions), heads * dim, dtype=x.dtype, device=DEV)
        out = torch.empty_like(q)
        kernels.kv8_write(xg, pos, torch.tensor(slots, dtype=torch.int32, device=DEV), cg, sg, *gpu, q, heads, kv_heads, dim, page,
                          status)
        row, tiles, items = 0, [], []
        for s, (a, n) in segments:
            if n > 1:
                tiles += [(s, row + i, min(128, n - i)) for i in range(0, n, 128)]
            else:
                items.append((row, s, a + 1, 0))
            row += n
        if tiles:
            seq, tok, rows = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in zip(*tiles))
            kernels.kv8_attn_prefill(q, q.stride(0), *gpu, tg, seq, tok, rows, pos, out, len(tiles), heads, kv_heads, dim, page, 0, scale)
        if items:
            kernels.kv8_attn_decode(q, q.stride(0), *gpu, tg, torch.tensor(items, dtype=torch.int32, device=DEV), work, out, len(items),
                                    heads, kv_heads, dim, page, 0, scale)
        compare(out, q, segments)
        for s, (a, n) in segments:
            at[s] += n
    # steps of single tokens, replayed: contexts and rows are in device memory
    xg = torch.zeros(2, width, dtype=DT[dtype], device=DEV)
    items = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    out = torch.zeros(2, heads * dim, dtype=DT[dtype], device=DEV)

    def step():
        kernels.kv8_attn_decode_rope(xg, xg.stride(0), *gpu, tg, items, work, out, 2, heads, kv_heads, dim, page, 0, scale, cg, sg,
                                     status)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(page + 2):
        x = torch.randn(2, width, generator=g).to(DT[dtype])
        xg.copy_(x)
        items.copy_(torch.tensor([(s, s, at[s] + 1, 0) for s in range(2)], dtype=torch.int32))
        graph.replay()
        slots = [int(table[s, at[s] // page]) * page + at[s] % page for s in range(2)]
        f = x.float()
        q = P.rotate(f[:, :heads * dim].view(2, heads, dim), cos[at], sin[at])
        P.store(P.rotate(f[:, heads * dim:-kv_heads * dim].view(2, kv_heads, dim), cos[at], sin[at]), slots, cache[0], cache[2])
        P.store(f[:, -kv_heads * dim:].reshape(2, kv_heads, dim), slots, cache[1], cache[3])
        for got, want in zip(gpu, cache):
            mask = table.flatten().long()
            assert torch.equal(got.view(torch.uint8).cpu()[mask], want[mask])
        compare(out, q, [(s, (at[s], 1)) for s in range(2)])
        at = [a + 1 for a in at]
    assert status.item() == 0


def test_on_another_stream():
    heads, kv_heads, dim, page = 4, 2, 64, 16
    ctxs = (300, 20)
    cache, table = filled(ctxs, heads, kv_heads, dim, page, seed=1)
    q = torch.randn(2, heads * dim).bfloat16().to(DEV)
    here = decode(q, on_gpu(cache), table, ctxs, heads, kv_heads, dim, page, 0, 0.125)
    gpu = on_gpu(cache)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        there = decode(q, gpu, table, ctxs, heads, kv_heads, dim, page, 0, 0.125)
    side.synchronize()
    assert torch.equal(here, there)


def test_the_cuda_core_kernel_first():
    """A process whose first portion goes to the CUDA cores, and its second to the tensor cores: each kernel's shared memory is asked for."""
    code = """
import sys, torch
sys.path.insert(0, "tests")
import test_kv8_gpu as T
from redline_b200.ops import kernels
cache, table = T.filled([130], 4, 2, 64, 16, seed=1)
gpu = T.on_gpu(cache)
q = torch.randn(130, 256, dtype=torch.bfloat16, device="cuda")
seq, tok, rows = T.tiles_of([(0, 130)])
pos = torch.arange(130, dtype=torch.int32, device="cuda")
outs = []
for impl in (1, 3, 0):
    outs.append(torch.empty_like(q))
    kernels.kv8_attn_prefill(q, 256, *gpu, table.to("cuda"), seq, tok, rows, pos, outs[-1], len(seq), 4, 2, 64, 16, 0, 0.125, impl=impl)
torch.cuda.synchronize()
assert all(torch.isfinite(o).all() for o in outs) and torch.equal(outs[1], outs[2])
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], cwd=root, check=True, timeout=300)
