"""Performance cases of the cache that is held in 8 bits: its write, and the attention that reads it.

The cache holds keys and values as e4m3 numbers in pages of 16, 32 or 64 tokens, and for every page and kv head one scale for
the keys and one for the values, a power of two (e8m0).  A block of values x (a page of one head) is stored as
x / 2^e rounded to e4m3, 2^e the smallest power of two for which the largest magnitude of the block is at most 448 * 2^e.
A page is filled in order: its first token sets the scale anew, a later one may raise it, and what lies in the page
before that token is then rescaled (exact but for numbers that fall below e4m3's normal range).

Four kinds of case:

  write   rotates q and k of a step's tokens (sequences with any number of new tokens) and stores k and v
  decode  one query token a sequence over its pages
  step    the same from the projection's unrotated rows: the token's own key and value are stored first
  prompt  portions of prompts, up to 128 query rows a tile, over the pages of their sequences

Sizes are those of this repository's configurations (head layouts 32/8/64, 32/8/128, 4/2/64, 3/1/128 and others), contexts
from one token to 131,072.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
TILE_ROWS = 128


def listed():
    def case(name, kind, heads, kv_heads, dim, page, dtype, seqs, ctx, new, window=0, mix=1):
        return {"name": name, "kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype,
                "seqs": seqs, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "new_lo": new[0], "new_hi": new[1], "window": window,
                "mix": mix}

    return [
        # the write of a step of eight single tokens, somewhere within their pages: latency alone
        case("write 8 single tokens", "write", 32, 8, 64, 16, "bf16", 8, (500, 4096), (1, 1)),
        # the write of one whole prompt of the benchmark's length
        case("write prompt 2048", "write", 32, 8, 64, 16, "bf16", 1, (0, 0), (2048, 2048)),
        # a mixed step: portions of odd lengths that begin within pages, beside single tokens, larger heads and pages
        case("write mixed portions", "write", 32, 8, 128, 32, "bf16", 9, (0, 900), (1, 700), mix=5),
        # a chat at batch one, its context just past 512
        case("step 1 x 513", "step", 32, 8, 64, 16, "bf16", 1, (513, 513), (1, 1)),
        # the benchmark's decode step: eight sequences near 4,096
        case("step 8 x 4096", "step", 32, 8, 64, 16, "bf16", 8, (3900, 4096), (1, 1)),
        # many short sequences
        case("step 64 x 516 to 768", "step", 32, 8, 64, 16, "bf16", 64, (516, 768), (1, 1)),
        # sequences of very different lengths under continuous batching, heads of 128, pages of 64
        case("decode 24 ragged", "decode", 32, 8, 128, 64, "bf16", 24, (64, 8192), (1, 1), mix=2),
        # one document of 131,072 tokens
        case("decode 1 x 131072", "decode", 32, 8, 128, 16, "bf16", 1, (131072, 131072), (1, 1)),
        # an odd portion of a prompt behind what the conversation has cached already
        case("prompt 333 behind 1000", "prompt", 32, 8, 64, 16, "bf16", 1, (1000, 1000), (333, 333)),
        # the fourth full portion of a long prompt
        case("prompt 2048 behind 6144", "prompt", 32, 8, 64, 16, "bf16", 1, (6144, 6144), (2048, 2048)),
        # heads of 128, three sequences of a batch at once
        case("prompt 3 portions, heads of 128", "prompt", 32, 8, 128, 16, "bf16", 3, (0, 2000), (300, 900), mix=3),
        # the 32-bit engine's small prompts, one kv head under three heads
        case("prompt float32", "prompt", 3, 1, 128, 16, "f32", 4, (0, 100), (33, 129), mix=4),
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["write", "decode", "step", "step", "prompt", "prompt"])
    heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 64), (32, 8, 128), (32, 8, 128), (4, 2, 64), (3, 1, 128),
                                       (20, 4, 128), (16, 1, 128), (8, 8, 64), (10, 2, 80), (12, 4, 96), (8, 1, 256)])
    dtype = "f32" if rng.random() < 0.2 else "bf16"
    page = rng.choice([16, 16, 32, 64])
    window = log_int(16, 2048) if rng.random() < 0.2 else 0
    size = kv_heads * dim
    if kind == "write":
        seqs = log_int(1, 64)
        hi = log_int(1, max(1, 4096 // seqs))
        new, ctx = (1 if rng.random() < 0.5 else hi, hi), (0, log_int(1, 1000))
        window = 0
    elif kind == "prompt":
        seqs = log_int(1, 6)
        most = 512 if dtype == "f32" or dim not in (64, 128) else 2048
        hi = max(2, log_int(2, most) // seqs)
        new = (max(2, hi // rng.choice([1, 2, 4])), hi)
        ctx = (0, log_int(1, 512 if most == 512 else 6000 if heads * dim <= 2048 else 2000))
    else:
        seqs = log_int(1, 128)
        most = min(131072, 120_000_000 // (2 * size * seqs))
        hi = log_int(1, max(1, most))
        ctx, new = (max(1, hi // rng.choice([1, 1, 4, 64])), hi), (1, 1)
    return {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "seqs": seqs,
            "ctx_lo": ctx[0], "ctx_hi": ctx[1], "new_lo": new[0], "new_hi": new[1], "window": window,
            "mix": rng.randrange(1 << 20)}


def lengths(case):
    """(cached tokens before the step, new tokens) of every sequence; the case's alone, whatever the seed.  In the kinds
    "decode" and "step" the context counts the query's own token."""
    r = random.Random(case["mix"])
    single = case["kind"] in ("decode", "step")
    got = []
    for _ in range(case["seqs"]):
        start, n = r.randint(case["ctx_lo"], case["ctx_hi"]), r.randint(case["new_lo"], case["new_hi"])
        got.append((max(start - 1, 0), 1) if single else (start, n))
    return got


def work(case):
    heads, kv_heads, dim, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    elem = 2 if case["dtype"] == "bf16" else 4
    tokens = pairs = keys = 0
    for start, n in lengths(case):
        tokens += n
        first = max(0, start + 1 - window) if window else 0
        keys += start + n - first
        for_all = n * start + n * (n + 1) // 2
        if window:
            # row i of the portion sees min(start + i + 1, window) keys
            short = max(0, min(n, window - start))
            for_all = short * start + short * (short + 1) // 2 + (n - short) * window
        pairs += for_all
    if case["kind"] == "write":
        return {"bytes": tokens * dim * ((2 * heads + 2 * kv_heads) * elem + 2 * kv_heads), "flops": 3.0 * tokens * dim * (heads + kv_heads)}
    cached = 2 * keys * kv_heads * dim + 2 * kv_heads * keys / case["page"]
    rows = 2 * tokens * heads * dim * elem
    if case["kind"] == "step":
        rows += 2 * tokens * kv_heads * dim * elem
    return {"bytes": cached + rows, "flops": 4.0 * pairs * heads * dim}


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    kind, page, dim = case["kind"], case["page"], case["dim"]
    heads, kv_heads, dtype = case["heads"], case["kv_heads"], TYPES[case["dtype"]]
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    segments = lengths(case)
    seqs = len(segments)
    blocks = [-(-(start + n) // page) for start, n in segments]
    width, pages = max(blocks), sum(blocks) + 1           # page 0 belongs to nobody
    order = (torch.randperm(pages - 1, generator=gen, device=DEVICE) + 1).cpu()
    table = torch.zeros((seqs, width), dtype=torch.int32)
    at = 0
    for s, b in enumerate(blocks):
        table[s, :b] = order[at:at + b]
        at += b
    position, slot, tile = [], [], []
    row = 0
    for s, (start, n) in enumerate(segments):
        p = torch.arange(start, start + n)
        position.append(p)
        slot.append(table[s].long()[p // page] * page + p % page)
        tile += [(s, row + i, min(TILE_ROWS, n - i)) for i in range(0, n, TILE_ROWS)]
        row += n
    tokens = row
    tile = torch.tensor(tile, dtype=torch.int32).t().contiguous().to(DEVICE)
    longest = max(n for _, n in segments)
    # row i of sequence s in a padded batch, and back (for whoever works on a padded batch)
    starts = torch.tensor([sum(n for _, n in segments[:s]) for s in range(seqs)])
    counts = torch.tensor([n for _, n in segments])
    step = torch.arange(longest)
    padded = torch.where(step[None] < counts[:, None], starts[:, None] + step[None], torch.full((1, 1), -1))
    context = torch.tensor([start + n for start, n in segments])
    items = torch.zeros((seqs, 4), dtype=torch.int32)
    items[:, 0] = starts
    items[:, 1] = torch.arange(seqs)
    items[:, 2] = context

    # keys of heads whose entries differ in size, values less so; what lies behind a sequence's end is what an earlier owner of
    # the page has left there
    def block(spread):
        x = torch.randn((pages, kv_heads, page, dim), generator=gen, device=DEVICE)
        size = torch.exp2(torch.randn((1, kv_heads, 1, dim), generator=gen, device=DEVICE) * spread)
        x = x * size * torch.exp2(torch.randn((pages, 1, 1, 1), generator=gen, device=DEVICE) * 0.3)
        mant, exp = torch.frexp(x.abs().amax((2, 3)))
        code = exp - 9 + (mant > 0.875).int()
        data = (x * power_of_two(-code)[:, :, None, None]).to(E4M3)
        return data, (code + 127).to(torch.uint8).view(E8M0)

    kcache, kscale = block(0.6)
    vcache, vscale = block(0.2)
    columns = (heads + 2 * kv_heads) * dim if kind in ("write", "step") else heads * dim
    x = torch.randn((tokens, columns), generator=gen, device=DEVICE)
    x[:, heads * dim:] *= 1.0 + torch.rand((1, columns - heads * dim), generator=gen, device=DEVICE)
    x = x.to(dtype)
    half = torch.arange(dim // 2, dtype=torch.float64, device=DEVICE)
    inv_freq = (500000.0 ** (-2.0 * half / dim)).float()
    angle = (torch.arange(int(context.max()), dtype=torch.float32, device=DEVICE)[:, None] * inv_freq).double()
    state = {
        "case": case, "x": x, "kcache": kcache, "vcache": vcache, "kscale": kscale, "vscale": vscale,
        "positions": torch.cat(position).int().to(DEVICE), "slots": torch.cat(slot).int().to(DEVICE),
        "table": table.to(DEVICE), "items": items.to(DEVICE), "tile_seq": tile[0], "tile_tok": tile[1], "tile_rows": tile[2],
        "padded": padded.to(DEVICE), "context": context.to(DEVICE),
        "cos": torch.cos(angle).float().contiguous(), "sin": torch.sin(angle).float().contiguous(),
        "status": torch.zeros(1, dtype=torch.int32, device=DEVICE), "max_ctx": int(context.max()), "sum_ctx": int(context.sum()),
        "tokens": tokens, "out": torch.empty((tokens, heads * dim), dtype=dtype, device=DEVICE), "kept": {},
    }
    return state


# --------------------------------------------------------------- plain form

def rotated(x, cos, sin):
    """Entry i with entry i + half, in 32 bits."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def power_of_two(e):
    """2^e for whole e, by its bits (0 below the normal numbers)."""
    return ((e + 127).clamp(min=0) << 23).int().view(torch.float32)


def stored(x, slots, cache, scale):
    """x [tokens, kv heads, dim] into the pages of ``slots``; the cache and its scales are updated in place."""
    page = cache.shape[2]
    at, off = (slots // page).long(), (slots % page).long()
    pages, kv_heads = scale.shape
    largest = torch.zeros((pages, kv_heads), device=x.device).scatter_reduce(
        0, at[:, None].expand(-1, kv_heads), x.abs().amax(-1), "amax")
    first = torch.full((pages,), page, device=x.device).scatter_reduce(0, at, off, "amin")
    mant, exp = torch.frexp(largest)
    code = torch.where(largest > 0, exp - 9 + (mant > 0.875).int() + 127, torch.ones_like(exp)).clamp(1, 246)
    before = scale.view(torch.uint8).int()
    after = torch.where((first == 0)[:, None], code, torch.maximum(code, before))
    touched = first < page
    after = torch.where(touched[:, None], after, before)
    down = power_of_two(before - after)
    row = torch.arange(page, device=x.device)
    old = cache.float()
    raised = (touched[:, None] & (row[None] < first[:, None]))[:, None, :, None] & (after > before)[:, :, None, None]
    new = torch.where(raised, old * down[:, :, None, None], old).to(E4M3)
    cache.copy_(new)
    unit = power_of_two(127 - after)[at]
    cache.view(torch.uint8)[at, :, off] = (x * unit[..., None]).to(E4M3).view(torch.uint8)
    scale.view(torch.uint8).copy_(after.to(torch.uint8))


def read(cache, scale, table):
    """The values that a sequence's pages stand for: [sequences, kv heads, keys, dim] in 32 bits."""
    got = cache.view(torch.uint8)[table.long()].view(E4M3).float() * scale.view(torch.uint8)[table.long()].view(E8M0).float()[..., None, None]
    seqs, blocks, kv_heads, page, dim = got.shape
    return got.permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, blocks * page, dim)


def attention(q, state):
    """q [tokens, heads, dim] in 32 bits over the pages; the result likewise."""
    case = state["case"]
    heads, kv_heads, dim, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    k = read(state["kcache"], state["kscale"], state["table"])
    v = read(state["vcache"], state["vscale"], state["table"])
    padded = state["padded"]
    seqs, rows = padded.shape
    live_row = padded >= 0
    position = state["positions"].long()[padded.clamp(min=0)]
    key = torch.arange(k.shape[2], device=k.device)
    seen = (key <= position[..., None]) & live_row[..., None]
    if window:
        seen &= key > position[..., None] - window
    grouped = q[padded.clamp(min=0)].view(seqs, rows, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    score = grouped @ k.transpose(-1, -2)[:, :, None] * (1.0 / math.sqrt(dim))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    del score
    total = weight.sum(-1, keepdim=True)
    v = torch.where((key[None] < state["context"][:, None])[:, None, :, None], v, torch.zeros_like(v))
    out = (weight @ v[:, :, None]) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, rows, heads, dim)
    return out[live_row]


def plain(state):
    case = state["case"]
    heads, kv_heads, dim, dtype = case["heads"], case["kv_heads"], case["dim"], state["x"].dtype
    kind, tokens = case["kind"], state["tokens"]
    x = state["x"].float()
    if kind in ("decode", "prompt"):
        return attention(x.view(tokens, heads, dim), state).reshape(tokens, -1).to(dtype)
    q, k, v = x.split([heads * dim, kv_heads * dim, kv_heads * dim], -1)
    at = state["positions"].long()
    cos, sin = state["cos"][at][:, None], state["sin"][at][:, None]
    q = rotated(q.view(tokens, heads, dim), cos, sin)
    stored(rotated(k.view(tokens, kv_heads, dim), cos, sin), state["slots"], state["kcache"], state["kscale"])
    stored(v.view(tokens, kv_heads, dim), state["slots"], state["vcache"], state["vscale"])
    caches = (state["kcache"], state["vcache"], state["kscale"], state["vscale"])
    if kind == "write":
        return (q.reshape(tokens, -1).to(dtype),) + caches
    return (attention(q, state).reshape(tokens, -1).to(dtype),) + caches


# ------------------------------------------------------------ the operators

def called(state):
    from redline_b200.ops import kernels

    case, s = state["case"], state
    heads, kv_heads, dim, page, window = case["heads"], case["kv_heads"], case["dim"], case["page"], case["window"]
    kind, x, out = case["kind"], s["x"], s["out"]
    scale = 1.0 / math.sqrt(dim)
    cache = (s["kcache"], s["vcache"], s["kscale"], s["vscale"])
    if kind == "write":
        kernels.kv8_write(x, s["positions"], s["slots"], s["cos"], s["sin"], *cache, out, heads, kv_heads, dim, page,
                          s["status"])
        return (out,) + cache
    if kind == "prompt":
        kernels.kv8_attn_prefill(x, x.stride(0), *cache, s["table"], s["tile_seq"], s["tile_tok"], s["tile_rows"],
                                 s["positions"], out, s["tile_seq"].numel(), heads, kv_heads, dim, page, window, scale)
        return out
    work = s["kept"].get("work")                     # a program keeps its workspace from step to step
    if work is None:
        work = s["kept"]["work"] = kernels.kv8_decode_workspace(len(s["items"]), heads, kv_heads, dim, x.device)
    if kind == "decode":
        kernels.kv8_attn_decode(x, x.stride(0), *cache, s["table"], s["items"], work, out, len(s["items"]), heads, kv_heads,
                                dim, page, window, scale, max_ctx=s["max_ctx"], sum_ctx=s["sum_ctx"])
        return out
    kernels.kv8_attn_decode_rope(x, x.stride(0), *cache, s["table"], s["items"], work, out, len(s["items"]), heads, kv_heads,
                                 dim, page, window, scale, s["cos"], s["sin"], s["status"], max_ctx=s["max_ctx"],
                                 sum_ctx=s["sum_ctx"])
    return (out,) + cache


def run(state):
    return called(state) if own else plain(state)


# ---------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    heads, kv_heads, dim, page, window = case["heads"], case["kv_heads"], case["dim"], case["page"], case["window"]
    kind = case["kind"]
    x = s["x"].double()
    half = dim // 2
    value = {"k": s["kcache"].double(), "v": s["vcache"].double()}
    power = {"k": s["kscale"].double(), "v": s["vscale"].double()}
    fp8 = {"k": s["kcache"].clone(), "v": s["vcache"].clone()}

    def turn(t, p):
        lo, hi = t[..., :half], t[..., half:]
        c, n = s["cos"].double()[p], s["sin"].double()[p]
        return torch.cat((lo * c - hi * n, lo * n + hi * c), -1)

    segments = lengths(case)
    powers = torch.tensor([2.0 ** e for e in range(-126, 120)], dtype=torch.float64, device=x.device)
    q = x[:, :heads * dim].reshape(-1, heads, dim)
    if kind in ("write", "step"):
        q = torch.stack([turn(q[:, h], s["positions"].long()) for h in range(heads)], 1)
        fresh = {"k": x[:, heads * dim:(heads + kv_heads) * dim], "v": x[:, (heads + kv_heads) * dim:]}
        for name, t in fresh.items():
            t = t.reshape(-1, kv_heads, dim)
            if name == "k":
                t = torch.stack([turn(t[:, h], s["positions"].long()) for h in range(kv_heads)], 1)
            row = 0
            for i, (start, n) in enumerate(segments):
                done = 0
                while done < n:
                    p = start + done
                    off = p % page
                    count = min(page - off, n - done)
                    block = int(s["table"][i, p // page])
                    part = t[row + done:row + done + count].transpose(0, 1)          # [kv heads, tokens, dim]
                    most = part.abs().amax((1, 2))
                    need = powers[torch.searchsorted(448.0 * powers, most)]          # the smallest with most <= 448 * need
                    unit = need if off == 0 else torch.maximum(need, power[name][block])
                    if off:
                        kept = value[name][block, :, :off] * (power[name][block] / unit)[:, None, None]
                        fp8[name][block, :, :off] = kept.float().to(E4M3)
                    fp8[name][block, :, off:off + count] = (part / unit[:, None, None]).float().to(E4M3)
                    power[name][block] = unit
                    value[name][block] = fp8[name][block].double()
                    done += count
                row += n
    caches = (value["k"], value["v"], power["k"], power["v"])
    if kind == "write":
        return (q.reshape(len(x), -1),) + caches
    out = torch.zeros((len(x), heads, dim), dtype=torch.float64, device=x.device)
    row = 0
    for i, (start, n) in enumerate(segments):
        end = start + n
        pages = s["table"][i, :-(-end // page)].long()
        for h in range(kv_heads):
            k = (value["k"][pages, h] * power["k"][pages, h][:, None, None]).reshape(-1, dim)[:end]
            v = (value["v"][pages, h] * power["v"][pages, h][:, None, None]).reshape(-1, dim)[:end]
            key = torch.arange(end, device=x.device)
            for r in range(0, n, 512):
                m = min(512, n - r)
                position = start + r + torch.arange(m, device=x.device)
                hide = key[None] > position[:, None]
                if window:
                    hide |= key[None] <= position[:, None] - window
                for g in range(h * heads // kv_heads, (h + 1) * heads // kv_heads):
                    logit = (q[row + r:row + r + m, g] @ k.T / math.sqrt(dim)).masked_fill(hide, -math.inf)
                    out[row + r:row + r + m, g] = torch.softmax(logit, -1) @ v
        row += n
    out = out.reshape(len(x), -1)
    return out if kind in ("decode", "prompt") else (out,) + caches
