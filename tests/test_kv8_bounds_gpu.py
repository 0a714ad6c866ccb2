"""The cache in 8 bits: what the calls do with entries of device memory that the host cannot check (page ids beyond
the pool, a sequence or a page under several items)."""

import math

import pytest
import torch

import plain_kv8 as P
from redline_b200.ops import kernels
from test_kv8_gpu import DEV, DT, angles, filled, near, on_gpu, tiles_of

pytestmark = pytest.mark.gpu
BAD = (0, 5, 2 ** 20, 2 ** 31 - 1, -1, -2 ** 31)      # (0: just beyond the pool)


def take_status():
    t = kernels.tc_status(torch.device(DEV, 0))
    code = t.item()
    t.zero_()
    return code


def bytes_of(cache):
    return [t.view(torch.uint8).cpu() for t in cache]


KINDS = [(4, 2, 64, 16, "bfloat16", 0), (4, 2, 64, 16, "bfloat16", 2), (4, 2, 64, 32, "bfloat16", 3), (4, 2, 64, 64, "bfloat16", 4),
         (3, 1, 128, 16, "bfloat16", 4), (3, 1, 128, 16, "bfloat16", 1), (4, 2, 64, 16, "float32", 0), (10, 2, 80, 16, "bfloat16", 0),
         (24, 2, 128, 32, "bfloat16", 2)]


def sequences(heads, kv_heads, dim, page, bad, poison):
    """Four sequences; one page of the second is ``bad`` (counted from the pool's end, or negative), the first and the last of the
    third as well."""
    ctxs = (100, 3 * page + 5, 4 * page, 40)
    cache, table = filled(ctxs, heads, kv_heads, dim, page, seed=dim + page, poison=poison)
    cache[0][0], cache[1][0], cache[2][0], cache[3][0] = 3, 5, 120, 121         # page 0 is finite here: its values are looked at
    pages = cache[0].shape[0]
    wrong = table.clone()
    for s, b in ((1, 1), (2, 0), (2, 3)):
        wrong[s, b] = bad if bad < 0 else min(pages + bad, 2 ** 31 - 1)
        table[s, b] = 0
    return ctxs, cache, table, wrong


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype,impl", KINDS)
def test_pages_beyond_the_pool_read_as_page_0(heads, kv_heads, dim, page, dtype, impl, bad):
    ctxs, cache, table, wrong = sequences(heads, kv_heads, dim, page, bad, True)
    gpu = on_gpu(cache)
    n, scale = len(ctxs), 1.0 / math.sqrt(dim)
    items = torch.tensor([(i, i, c, 0) for i, c in enumerate(ctxs)], dtype=torch.int32, device=DEV)
    work = kernels.kv8_decode_workspace(n, heads, kv_heads, dim, torch.device(DEV))
    q = torch.randn(n, heads * dim, generator=torch.Generator().manual_seed(1)).to(DT[dtype]).to(DEV)
    outs = []
    for t, code in ((table, 0), (wrong, 16), (table, 0)):
        out = torch.empty_like(q)
        kernels.kv8_attn_decode(q, q.stride(0), *gpu, t.to(DEV), items, work, out, n, heads, kv_heads, dim, page, 0, scale, impl=impl)
        assert take_status() == code
        outs.append(out)
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    assert all(torch.equal(a, b) for a, b in zip(bytes_of(gpu), cache))


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype,impl", KINDS)
def test_nothing_is_stored_beyond_the_pool(heads, kv_heads, dim, page, dtype, impl, bad):
    """The third sequence's newest page is bad, the second has a bad one behind its newest: the other tokens are stored, bit 4 tells."""
    ctxs, cache, table, wrong = sequences(heads, kv_heads, dim, page, bad, False)
    gpu = on_gpu(cache)
    n = len(ctxs)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(n, (heads + 2 * kv_heads) * dim, generator=g).to(DT[dtype])
    cos, sin = angles(300, dim)
    items = torch.tensor([(i, i, c, 0) for i, c in enumerate(ctxs)], dtype=torch.int32, device=DEV)
    work = kernels.kv8_decode_workspace(n, heads, kv_heads, dim, torch.device(DEV))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    xg, out = x.to(DEV), torch.empty(n, heads * dim, dtype=x.dtype, device=DEV)
    kernels.kv8_attn_decode_rope(xg, xg.stride(0), *gpu, wrong.to(DEV), items, work, out, n, heads, kv_heads, dim, page, 0,
                                 1.0 / math.sqrt(dim), cos.to(DEV), sin.to(DEV), status, impl=impl)
    assert status.item() == 4 and take_status() == 0
    at = [c - 1 for c in ctxs]
    slots = [int(table[s, p // page]) * page + p % page if s != 2 else -1 for s, p in enumerate(at)]
    k, v = x.float()[:, heads * dim:].split([kv_heads * dim] * 2, -1)
    P.store(P.rotate(k.reshape(n, kv_heads, dim), cos[at], sin[at]), slots, cache[0], cache[2])
    P.store(v.reshape(n, kv_heads, dim), slots, cache[1], cache[3])
    for got, want in zip(bytes_of(gpu), cache):
        assert torch.equal(got, want)
    assert (work[1] == 0).all()


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype,impl", [(4, 2, 64, 16, "bfloat16", 3), (3, 1, 128, 32, "bfloat16", 3),
                                                                (4, 2, 64, 16, "bfloat16", 1), (4, 2, 64, 64, "float32", 0),
                                                                (10, 2, 80, 16, "bfloat16", 0)])
def test_prompts_over_pages_beyond_the_pool(heads, kv_heads, dim, page, dtype, impl, bad):
    ctxs, cache, table, wrong = sequences(heads, kv_heads, dim, page, bad, True)
    gpu = on_gpu(cache)
    segments = [(c - min(c, 30), min(c, 30)) for c in ctxs]
    positions = torch.tensor([p for a, n in segments for p in range(a, a + n)], dtype=torch.int32, device=DEV)
    seq, tok, rows = tiles_of(segments)
    q = torch.randn(len(positions), heads * dim, generator=torch.Generator().manual_seed(1)).to(DT[dtype]).to(DEV)
    outs = []
    for t, code in ((table, 0), (wrong, 16)):
        out = torch.empty_like(q)
        kernels.kv8_attn_prefill(q, q.stride(0), *gpu, t.to(DEV), seq, tok, rows, positions, out, len(seq), heads, kv_heads, dim, page, 0,
                                 1.0 / math.sqrt(dim), impl=impl)
        assert take_status() == code
        outs.append(out)
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0], outs[1])


def fresh(n, blocks, heads, kv_heads, dim, page, dtype, seed=1, extra=0):
    """``n`` sequences of random finite pages and rows [q | k | v] for them."""
    g = torch.Generator().manual_seed(seed)
    pages = n * blocks + 1 + extra
    cache = [torch.randint(0, 126, (pages, kv_heads, page, dim), generator=g).to(torch.uint8) for _ in range(2)]
    cache += [torch.randint(115, 120, (pages, kv_heads), generator=g).to(torch.uint8) for _ in range(2)]
    table = (torch.randperm(n * blocks, generator=g) + 1).view(n, blocks).int()
    x = torch.randn(n, (heads + 2 * kv_heads) * dim, generator=g).to(DT[dtype])
    return cache, table, x


def stored(x, table, items, keep, cos, sin, cache, heads, kv_heads, dim, page):
    """The restatement's store of the items' tokens, of those that are kept."""
    at = [c - 1 for _, c in items]
    slots = [int(table[s, p // page]) * page + p % page if k else -1 for (s, _), p, k in zip(items, at, keep)]
    k, v = x.float()[:, heads * dim:].split([kv_heads * dim] * 2, -1)
    P.store(P.rotate(k.reshape(len(x), kv_heads, dim), cos[at], sin[at]), slots, cache[0], cache[2])
    P.store(v.reshape(len(x), kv_heads, dim), slots, cache[1], cache[3])


def rope(x, gpu, table, items, cos, sin, heads, kv_heads, dim, page, impl):
    n = len(items)
    info = torch.tensor([(i, s, c, 0) for i, (s, c) in enumerate(items)], dtype=torch.int32, device=DEV)
    work = kernels.kv8_decode_workspace(n, heads, kv_heads, dim, torch.device(DEV))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    xg, out = x.to(DEV), torch.empty(len(x), heads * dim, dtype=x.dtype, device=DEV)
    kernels.kv8_attn_decode_rope(xg, xg.stride(0), *gpu, table.to(DEV), info, work, out, n, heads, kv_heads, dim, page, 0,
                                 1.0 / math.sqrt(dim), cos.to(DEV), sin.to(DEV), status, impl=impl)
    assert (work[1] == 0).all()
    return out, status.item()


# items (sequence, context) and which of them are stored
TWICE = [([(0, 20), (1, 18), (1, 19), (2, 40)], (1, 1, 0, 1)),          # one sequence, places that follow one another
         ([(1, 64), (0, 20), (1, 65), (2, 40)], (1, 1, 0, 1)),          # one sequence, two pages
         ([(3, 20), (4, 25), (0, 9), (3, 70)], (1, 0, 1, 0)),           # two sequences that name one page; one of them once more
         ([(0, 0), (0, 33), (1, 1), (1, 1)], (0, 1, 1, 0))]             # (an item without keys stores nothing)


@pytest.mark.parametrize("items,keep", TWICE)
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype,impl", KINDS)
def test_a_sequence_or_a_page_twice(heads, kv_heads, dim, page, dtype, impl, items, keep):
    """Whichever kernel stores the tokens: the first is stored, the others are not, and bit 8 tells."""
    cache, table, x = fresh(5, 8, heads, kv_heads, dim, page, dtype)
    table[4] = table[3]
    x = x[:len(items)].contiguous()
    cos, sin = angles(300, dim)
    gpu = on_gpu(cache)
    _, code = rope(x, gpu, table, items, cos, sin, heads, kv_heads, dim, page, impl)
    assert code == 8
    stored(x, table, items, keep, cos, sin, cache, heads, kv_heads, dim, page)
    for got, want in zip(bytes_of(gpu), cache):
        assert torch.equal(got, want)


@pytest.mark.parametrize("twice", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype,impl", [(4, 2, 64, 16, "bfloat16", 0), (4, 2, 64, 16, "bfloat16", 3),
                                                                (4, 1, 128, 32, "bfloat16", 2), (2, 1, 64, 64, "bfloat16", 0),
                                                                (2, 1, 64, 16, "float32", 0), (2, 1, 80, 16, "bfloat16", 0)])
def test_more_items_than_a_launch_takes(heads, kv_heads, dim, page, dtype, impl, twice):
    """Several launches over one workspace: tokens stored, rows attended, a sequence of the first launch in the last once more."""
    n = 2100
    cache, table, x = fresh(n, 2, heads, kv_heads, dim, page, dtype)
    items = [(i, 1 + i * 7 % (2 * page)) for i in range(n)]
    keep = [1] * n
    if twice:
        items[2090], keep[2090] = (3, items[3][1] + 1), 0
    cos, sin = angles(2 * page + 2, dim)
    gpu = on_gpu(cache)
    out, code = rope(x, gpu, table, items, cos, sin, heads, kv_heads, dim, page, impl)
    assert code == (8 if twice else 0)
    stored(x, table, items, keep, cos, sin, cache, heads, kv_heads, dim, page)
    for got, want in zip(bytes_of(gpu), cache):
        assert torch.equal(got, want)
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    q = P.rotate(x.float()[:, :heads * dim].view(n, heads, dim), cos[[c - 1 for _, c in items]], sin[[c - 1 for _, c in items]])
    for i in (0, 1, 500, 1022, 1023, 1024, 1025, 1500, 2047, 2048, 2049, 2098, 2099):
        s, c = items[i]
        ref = P.attend(q[i:i + 1], k, v, table[s], [c - 1], 0, 1.0 / math.sqrt(dim))
        near(out[i].view(1, heads, dim), ref, v[table[s][:-(-c // page)].long()], dtype)


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [(4, 2, 64, 16, "float32"), (10, 2, 80, 16, "bfloat16"), (40, 2, 64, 64, "bfloat16")])
def test_a_refused_call_stores_nothing(heads, kv_heads, dim, page, dtype):
    cache, table, x = fresh(3, 4, heads, kv_heads, dim, page, dtype)
    cos, sin = angles(100, dim)
    gpu = on_gpu(cache)
    for impl in (2, 3, 4):
        with pytest.raises(kernels.KernelError):
            rope(x, gpu, table, [(0, 5), (1, 20), (2, 33)], cos, sin, heads, kv_heads, dim, page, impl)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(bytes_of(gpu), cache))


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype,n", [(4, 2, 64, 16, "bfloat16", 5), (3, 1, 128, 16, "bfloat16", 5), (32, 8, 64, 32, "bfloat16", 40),
                                                             (16, 8, 128, 16, "bfloat16", 40), (4, 2, 64, 16, "float32", 5), (10, 2, 80, 16, "bfloat16", 5)])
def test_tiles_without_rows(heads, kv_heads, dim, page, dtype, n):
    """Among the others, first and last, at positions that begin a key tile and others; a list of nothing else."""
    segments = [(128 * (s % 3) + s % 2, 1 + 29 * s % 120) for s in range(n)]
    lengths = [a + m for a, m in segments]
    cache, table = filled(lengths, heads, kv_heads, dim, page, seed=1)
    gpu = on_gpu(cache)
    positions = torch.tensor([p for a, m in segments for p in range(a, a + m)], dtype=torch.int32, device=DEV)
    seq, tok, rows = (t.tolist() for t in tiles_of(segments))
    full = list(zip(seq, tok, rows))
    with_empty = [(0, tok[0], 0)]
    for i, t in enumerate(full):
        with_empty += [t, (t[0], t[1], 0)] if i % 2 else [t]
    q = torch.randn(len(positions), heads * dim, generator=torch.Generator().manual_seed(1)).to(DT[dtype]).to(DEV)

    def run(tiles, out):
        lists = [torch.tensor(t, dtype=torch.int32, device=DEV) for t in zip(*tiles)]
        kernels.kv8_attn_prefill(q, q.stride(0), *gpu, table.to(DEV), *lists, positions, out, len(tiles), heads, kv_heads, dim, page, 0,
                                 1.0 / math.sqrt(dim))
        assert take_status() == 0
        return out

    want, got = run(full, torch.empty_like(q)), run(with_empty, torch.empty_like(q))
    assert torch.isfinite(want).all() and torch.equal(want, got)
    nothing = run([(0, 0, 0)] * 7, torch.full_like(q, 9.0))
    assert (nothing == 9.0).all()
