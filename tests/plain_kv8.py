"""The 8-bit cache restated with elementary operations: its format, its write, and attention over it in 64 bits.

A page of one kv head is page_size rows of e4m3 numbers and one scale 2^(code - 127); a block of values is stored as
x / 2^e rounded to e4m3, 2^e the smallest power of two with max |x| <= 448 * 2^e."""

from __future__ import annotations

import math
from typing import Optional

import torch

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def code_of(largest: float) -> int:
    """The scale's byte for a block whose largest finite magnitude is ``largest``."""
    if largest == 0.0:
        return 1
    code = 1
    while code < 246 and largest > 448.0 * 2.0 ** (code - 127):
        code += 1
    return code


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Entry i with entry i + half in float32, every product and sum rounded (x [T, heads, D], cos / sin [T, D/2])."""
    x, half = x.float(), x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def store(x: torch.Tensor, slots, cache: torch.Tensor, scale: torch.Tensor) -> None:
    """x [T, heads, D] float32 (on the CPU) to the slots of ``cache`` [pages, heads, page, D] (uint8 bytes) and ``scale``
    [pages, heads] (uint8), as kv8_write does it: run by run."""
    page_size = cache.shape[2]
    slots = [int(s) for s in slots]
    done = set()
    t = 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] >= cache.shape[0] * page_size:
            t += 1
            continue
        page, off = divmod(slots[t], page_size)
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and off + n < page_size:
            n += 1
        if page not in done:
            done.add(page)
            for h in range(cache.shape[1]):
                block = x[t:t + n, h]
                finite = torch.isfinite(block)
                largest = block[finite].abs().max().item() if finite.any() else 0.0
                code = code_of(largest)
                if off > 0:
                    old = min(int(scale[page, h]), 254)
                    if code > old:
                        kept = cache[page, h, :off].view(E4M3).float() * 2.0 ** max(old - code, -127)
                        cache[page, h, :off] = kept.to(E4M3).view(torch.uint8)
                    else:
                        code = old
                scale[page, h] = code
                unit = torch.tensor(2.0 ** (127 - code), dtype=torch.float64).float()
                y = (block * unit).clamp(-448.0, 448.0)
                y = torch.where(finite, y, torch.full_like(y, math.nan))
                cache[page, h, off:off + n] = y.to(E4M3).view(torch.uint8)
        t += n


def values(cache: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """What the cache stands for, [pages, heads, page, D] in float64."""
    exponent = scale.view(torch.uint8).double() - 127.0
    return cache.view(torch.uint8).view(E4M3).double() * torch.exp2(exponent)[..., None, None]


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table, positions, window: int, scale: float,
           pages: Optional[int] = None) -> torch.Tensor:
    """q [rows, heads, D] of one sequence over the pages ``table`` of k and v (values()), float64."""
    kv_heads, page = k.shape[1], k.shape[2]
    end = int(max(positions)) + 1
    table = [int(b) for b in table[:-(-end // page)]]
    keys = k[table].permute(1, 0, 2, 3).reshape(kv_heads, -1, k.shape[3])[:, :end]
    vals = v[table].permute(1, 0, 2, 3).reshape(kv_heads, -1, k.shape[3])[:, :end]
    out = torch.empty_like(q, dtype=torch.float64)
    group = q.shape[1] // kv_heads
    for i, p in enumerate(int(x) for x in positions):
        lo = max(0, p + 1 - window) if window else 0
        for h in range(q.shape[1]):
            kk, vv = keys[h // group, lo:p + 1], vals[h // group, lo:p + 1]
            w = torch.softmax(kk @ q[i, h].double() * scale, -1)
            out[i, h] = w @ vv
    return out
