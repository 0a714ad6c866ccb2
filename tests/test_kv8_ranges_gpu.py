"""Attention over the cache in 8 bits where numbers are not finite (what is not a number reaches the rows that see it and no others), or
far apart."""

import math

import pytest
import torch

import plain_kv8 as P
from redline_b200.ops import kernels
from test_kv8_gpu import DEV, DT, angles, filled, near, on_gpu, tiles_of

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
    (10, 2, 80, 16, 0, "bfloat16", 0), (2, 1, 16, 16, 25, "bfloat16", 0), (4, 2, 64, 16, 0, "bfloat16", 3), (3, 1, 128, 32, 0, "bfloat16", 3),
    (4, 2, 64, 64, 90, "bfloat16", 3), (5, 1, 128, 16, 60, "bfloat16", 3)])
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


def formula(q, k, v, table, positions, window, scale, dtype, rounded_q=False, times=None):
    """Attention of q [rows, heads, D] in float64 and a bound of each number's own.  With w_j the weights:

      |error| <= r |result| + (p + 2 d) sum_j w_j |v_j|
      r   the result's one rounding: 2^-8 (bfloat16), 2^-24 (float32)
      p   the weights' rounding and the sums': 2^-11 for halves, and 2^-16 (chains of up to a few thousand terms in float32)
      d   the largest error of a score, which moves weights by a factor of 1 + d and the denominator likewise: of the products' sums in
          float32 2^-17 of sum_d |q_d k_d| (128 roundings of 2^-24), and 2^-11 more where q is rounded to halves on its way (``rounded_q``)

    times: how often each key counts (for tests of the bound itself)."""
    heads, kv_heads, page = q.shape[1], k.shape[1], k.shape[2]
    end = int(max(positions)) + 1
    dev = k.device
    blocks = table[:-(-end // page)].long().to(dev)
    keys = k[blocks].permute(1, 0, 2, 3).reshape(kv_heads, -1, k.shape[3])[:, :end]
    vals = v[blocks].permute(1, 0, 2, 3).reshape(kv_heads, -1, k.shape[3])[:, :end]
    keys, vals = (t.repeat_interleave(heads // kv_heads, 0) for t in (keys, vals))      # [heads, keys, D]
    qd = q.to(dev).double().transpose(0, 1)
    score, size = qd @ keys.transpose(1, 2) * scale, qd.abs() @ keys.abs().transpose(1, 2) * scale
    at, key = torch.tensor(list(positions), device=dev), torch.arange(end, device=dev)
    hide = key[None] > at[:, None]
    if window:
        hide |= key[None] <= at[:, None] - window
    if times is not None:
        score = score + torch.log(times.to(dev))
    w = torch.softmax(score.masked_fill(hide, -math.inf), -1)
    ref, spread = (w @ vals).transpose(0, 1), (w @ vals.abs()).transpose(0, 1)
    d = size.masked_fill(hide, 0).amax(-1).transpose(0, 1)[..., None] * (2.0 ** -17 + (2.0 ** -11 if rounded_q else 0.0))
    r, p = (2.0 ** -24, 2.0 ** -16) if dtype == "float32" else (2.0 ** -8, 2.0 ** -11 + 2.0 ** -16)
    return ref, r * ref.abs() + (p + 2 * d) * spread


def tight(out, q, k, v, table, positions, window, scale, dtype, rounded_q=False):
    """``out`` [rows, heads, D] within the formula's bound."""
    ref, limit = formula(q, k.to(out.device), v.to(out.device), table, positions, window, scale, dtype, rounded_q)
    assert torch.isfinite(out).all()
    err = (out.double() - ref).abs()
    assert (err <= limit).all(), f"{(err / limit.clamp(min=1e-300)).max().item():.2f} of the limit"


def magnitudes(lengths, kv_heads, dim, page, kexp, vexp, seed):
    """``filled`` with keys of sequence s times 2^kexp[s], values times 2^vexp[s] (an exponent of a block moves its scale alone)."""
    cache, table = filled(lengths, kv_heads, kv_heads, dim, page, seed=seed)
    for s, n in enumerate(lengths):
        mine = table[s][:-(-n // page)].long()
        cache[2][mine] = (cache[2][mine].int() + kexp[s]).to(torch.uint8)
        cache[3][mine] = (cache[3][mine].int() + vexp[s]).to(torch.uint8)
    return cache, table


@pytest.mark.parametrize("heads,kv_heads,dim,page,impl", [(4, 2, 64, 16, 3), (3, 1, 64, 32, 3), (4, 2, 128, 16, 3), (4, 2, 64, 16, 1),
                                                          (10, 2, 80, 16, 0)])
def test_prompts_of_queries_of_any_size(heads, kv_heads, dim, page, impl):
    """Queries beyond what a half holds and far below it, over keys that make up for it; rows of other sizes beside them in a tile."""
    qexp = (0, 17, 40, 100, -17, -40, -90, 110)
    segments = tuple((20 * s, 70 + s) for s in range(len(qexp))) + ((0, 300),)
    lengths = [a + n for a, n in segments]
    cache, table = magnitudes(lengths, kv_heads, dim, page, [-e for e in qexp] + [0], [0, 60, -60, 90, 0, -90, 30, 0, 0], dim)
    g = torch.Generator().manual_seed(5)
    q = [torch.randn(n, heads * dim, generator=g) * 2.0 ** e for (_, n), e in zip(segments, qexp + (0,))]
    q[-1] *= torch.exp2(-torch.randint(0, 120, (len(q[-1]), 1), generator=g).float())     # (every row its own size, down to all keys alike)
    q[0][3] = 0.0
    q = torch.cat(q).bfloat16()
    scale = 1.0 / math.sqrt(dim)
    out = prefill(q, on_gpu(cache), table, segments, heads, kv_heads, dim, page, 0, scale, impl)
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    row = 0
    for s, (a, n) in enumerate(segments):
        tight(out[row:row + n].view(n, heads, dim), q[row:row + n].view(n, heads, dim), k, v, table[s], range(a, a + n), 0, scale, "bfloat16")
        row += n


def test_prompts_of_queries_that_are_not_finite():
    """Make their own rows not a number, and no others."""
    heads, kv_heads, dim, page, n = 4, 2, 64, 16, 200
    cache, table = filled((n,), heads, kv_heads, dim, page, seed=1)
    q = torch.randn(n, heads * dim, generator=torch.Generator().manual_seed(1)).bfloat16()
    q[50, 3], q[60, dim + 5], q[130, 2 * dim] = math.inf, math.nan, -math.inf
    outs = [prefill(q, on_gpu(cache), table, ((0, n),), heads, kv_heads, dim, page, 0, 0.125, impl).view(n, heads, dim) for impl in (1, 3)]
    nan = torch.zeros(n, heads, dim, dtype=torch.bool)
    nan[50, 0] = nan[60, 1] = nan[130, 2] = True
    for out in outs:
        assert torch.equal(torch.isnan(out).cpu(), nan) and torch.isfinite(out[~nan.to(out.device)]).all()


@pytest.mark.parametrize("dim,impl", [(64, 3), (128, 3), (64, 1)])
def test_prompts_of_many_small_weights(dim, impl):
    """One key takes nearly all the weight and its value is nothing: what is left are thousands of keys of one small weight each."""
    heads, kv_heads, page, n, past = 2, 1, 16, 130, 4000
    cache, table = filled((past + n,), heads, kv_heads, dim, page, seed=2)
    k, v = torch.zeros(past + n, kv_heads, dim), torch.ones(past + n, kv_heads, dim)
    v *= 1.0 + torch.randint(0, 4, (past + n, 1, 1), generator=torch.Generator().manual_seed(1)) / 4.0
    k[0, 0, 0], v[:16] = 1.0, 0.0
    slot = [int(table[0, p // page]) * page + p % page for p in range(past + n)]
    P.store(k, slot, cache[0], cache[2])
    P.store(v, slot, cache[1], cache[3])
    q = torch.zeros(n, heads, dim)
    q[:, :, 0] = (torch.arange(n)[:, None] * 0.15 + torch.tensor([0.0, 0.07])) * math.log(2.0)      # weights from 1 to 2^-19.4 of the one key's
    q = q.view(n, -1).bfloat16()
    out = prefill(q, on_gpu(cache), table, ((past, n),), heads, kv_heads, dim, page, 0, 1.0, impl)
    kd, vd = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    tight(out.view(n, heads, dim), q.view(n, heads, dim), kd, vd, table[0], range(past, past + n), 0, 1.0, "bfloat16")


FAR = [(4, 2, 64, 16, 0, "bfloat16", 3), (3, 1, 128, 16, 0, "bfloat16", 3), (4, 2, 64, 32, 100, "bfloat16", 3), (4, 2, 64, 16, 0, "bfloat16", 1),
       (4, 2, 64, 16, 0, "float32", 0), (10, 2, 80, 16, 0, "bfloat16", 0)]


@pytest.mark.parametrize("far", [5, 20, 22, 23, 30, 60])
@pytest.mark.parametrize("heads,kv_heads,dim,page,window,dtype,impl", FAR)
def test_prompts_over_pages_far_apart(heads, kv_heads, dim, page, window, dtype, impl, far):
    """Pages that only later rows of a tile see are 2^far larger, and queries are such that scores are of any one size; pages of all
    sizes behind one another; every row right by its own measure."""
    segments = ((0, 260), (100, 180), (0, 90))
    lengths = [a + n for a, n in segments]
    cache, table = filled(lengths, heads, kv_heads, dim, page, seed=dim + far)
    small = 64 // page
    for b, p in enumerate(table[0].tolist()):
        if p and b < small:
            cache[2][p] -= far
            cache[3][p] -= far
    for b, p in enumerate(table[1].tolist()):
        if p:
            cache[3][p] = (cache[3][p].int() + (-far, 0, far, 3, -far // 2)[b % 5]).to(torch.uint8)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(sum(n for _, n in segments), heads * dim, generator=g)
    q[:64] *= 2.0 ** far
    q = q.to(DT[dtype])
    scale = 1.0 / math.sqrt(dim)
    out = prefill(q, on_gpu(cache), table, segments, heads, kv_heads, dim, page, window, scale, impl)
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    row = 0
    for s, (a, n) in enumerate(segments):
        tight(out[row:row + n].view(n, heads, dim), q[row:row + n].view(n, heads, dim), k, v, table[s], range(a, a + n), window, scale, dtype)
        row += n


def test_prompts_of_very_many_items_far_apart():
    """More of them to a CTA than it keeps a list of."""
    heads = kv_heads = 32
    dim, page, n = 64, 16, 300
    segments = ((15, 2),) * n
    cache, table = filled((17,) * n, heads, kv_heads, dim, page, seed=3)
    cache[3][table[:, 0].long()] -= 40
    q = torch.randn(2 * n, heads * dim, generator=torch.Generator().manual_seed(6)).bfloat16()
    out = prefill(q, on_gpu(cache), table, segments, heads, kv_heads, dim, page, 0, 0.125, 3)
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    for s in (0, 1, 77, 150, 298, 299):
        tight(out[2 * s:2 * s + 2].view(2, heads, dim), q[2 * s:2 * s + 2].view(2, heads, dim), k, v, table[s], (15, 16), 0, 0.125, "bfloat16")


def test_a_page_of_zeros_is_not_far_from_any():
    """Its scale is the smallest there is."""
    heads, kv_heads, dim, page, n = 4, 2, 64, 16, 200
    cache, table = filled((n,), heads, kv_heads, dim, page, seed=3)
    for b in (0, 3, 7):
        p = int(table[0, b])
        cache[0][p], cache[1][p], cache[2][p], cache[3][p] = 0, 0, 1, 1
    q = torch.randn(n, heads * dim, generator=torch.Generator().manual_seed(6)).bfloat16()
    out = prefill(q, on_gpu(cache), table, ((0, n),), heads, kv_heads, dim, page, 0, 0.125, 3)
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    tight(out.view(n, heads, dim), q.view(n, heads, dim), k, v, table[0], range(n), 0, 0.125, "bfloat16")


def decode(q, gpu, table, ctxs, heads, kv_heads, dim, page, window, scale, impl):
    n = len(ctxs)
    items = torch.tensor([(i, i, c, 0) for i, c in enumerate(ctxs)], dtype=torch.int32, device=DEV)
    work = kernels.kv8_decode_workspace(n, heads, kv_heads, dim, torch.device(DEV))
    qg, out = q.to(DEV), torch.empty(n, heads * dim, dtype=q.dtype, device=DEV)
    kernels.kv8_attn_decode(qg, qg.stride(0), *gpu, table.to(DEV), items, work, out, n, heads, kv_heads, dim, page, window, scale, impl=impl)
    assert (work[1] == 0).all()
    return out


SINGLE = [(4, 2, 64, 16, "bfloat16"), (16, 1, 64, 32, "bfloat16"), (3, 1, 128, 16, "bfloat16"), (16, 1, 128, 64, "bfloat16"),
          (4, 2, 64, 16, "float32"), (10, 2, 80, 16, "bfloat16")]


@pytest.mark.parametrize("far", [5, 10, 11, 30, 60])
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SINGLE)
@pytest.mark.parametrize("impl", [0, 1, 2, 3, 4])
def test_single_tokens_over_pages_far_apart(heads, kv_heads, dim, page, dtype, impl, far):
    """Values of pages 2^far apart: the large ones under weights that are next to nothing, and all sizes behind one another."""
    if impl and (dtype == "float32" or dim == 80):
        pytest.skip("one way only")
    ctxs = (300, 1500, 64, 200, 900)
    cache, table = filled(ctxs, heads, kv_heads, dim, page, seed=far)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(len(ctxs), heads, dim, generator=g)
    for s, n in enumerate(ctxs):
        for b, p in enumerate(table[s].tolist()):
            if not p:
                continue
            if s % 2:                            # every size, the token's own page among them
                cache[3][p] = (cache[3][p].int() + (0, -far, far, 2, -far // 2)[b % 5]).to(torch.uint8)
            elif b == 1:                         # one page of large values, its keys turned away from q
                cache[3][p] += far
                away = -q[s].view(kv_heads, heads // kv_heads, dim).sum(1) * (far * math.log(2.0) * 1.5 * math.sqrt(dim) / dim)
                bytes_, scales = torch.zeros_like(cache[0][:1]), torch.zeros_like(cache[2][:1])
                P.store(away[None].expand(page, -1, -1), range(page), bytes_, scales)
                cache[0][p], cache[2][p] = bytes_[0], scales[0]
    q = q.view(len(ctxs), -1).to(DT[dtype])
    scale = 1.0 / math.sqrt(dim)
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    for window in (0, 100):
        out = decode(q, on_gpu(cache), table, ctxs, heads, kv_heads, dim, page, window, scale, impl)
        for s, n in enumerate(ctxs):
            tight(out[s].view(1, heads, dim), q[s].view(1, heads, dim), k, v, table[s], [n - 1], window, scale, dtype)


@pytest.mark.parametrize("heads,kv_heads,dim,page,impl", [(4, 2, 64, 16, 2), (4, 2, 64, 32, 3), (3, 1, 128, 16, 4), (16, 1, 128, 32, 2),
                                                          (4, 2, 64, 64, 2)])
def test_tokens_stored_beside_pages_far_apart(heads, kv_heads, dim, page, impl):
    """The token's own value far larger, or far smaller, than what the sequence holds: stored bit for bit, attended by its own measure."""
    ctxs = (100, 130, 65, 200, 49, 33)
    cache, table = filled(ctxs, heads, kv_heads, dim, page, seed=7, poison=False)
    g = torch.Generator().manual_seed(3)
    n = len(ctxs)
    x = torch.randn(n, (heads + 2 * kv_heads) * dim, generator=g)
    x[:, (heads + kv_heads) * dim:] *= 2.0 ** torch.tensor([40.0, -40.0, 12.0, -12.0, 90.0, 0.0])[:, None]
    x = x.bfloat16()
    cos, sin = angles(300, dim)
    gpu = on_gpu(cache)
    items = torch.tensor([(i, i, c, 0) for i, c in enumerate(ctxs)], dtype=torch.int32, device=DEV)
    work = kernels.kv8_decode_workspace(n, heads, kv_heads, dim, torch.device(DEV))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    xg, out = x.to(DEV), torch.empty(n, heads * dim, dtype=x.dtype, device=DEV)
    scale = 1.0 / math.sqrt(dim)
    kernels.kv8_attn_decode_rope(xg, xg.stride(0), *gpu, table.to(DEV), items, work, out, n, heads, kv_heads, dim, page, 0, scale,
                                 cos.to(DEV), sin.to(DEV), status, impl=impl)
    at = [c - 1 for c in ctxs]
    slots = [int(table[s, p // page]) * page + p % page for s, p in enumerate(at)]
    f = x.float()
    P.store(P.rotate(f[:, heads * dim:-kv_heads * dim].reshape(n, kv_heads, dim), cos[at], sin[at]), slots, cache[0], cache[2])
    P.store(f[:, -kv_heads * dim:].reshape(n, kv_heads, dim), slots, cache[1], cache[3])
    for got, want in zip(gpu, cache):
        assert torch.equal(got.view(torch.uint8).cpu(), want)
    assert status.item() == 0
    k, v = P.values(cache[0], cache[2]), P.values(cache[1], cache[3])
    q = P.rotate(f[:, :heads * dim].view(n, heads, dim), cos[at], sin[at])
    for s, c in enumerate(ctxs):
        tight(out[s].view(1, heads, dim), q[s:s + 1], k, v, table[s], [c - 1], 0, scale, "bfloat16", rounded_q=True)
