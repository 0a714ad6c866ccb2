"""Device memory of the cache: per group ONE allocation, zero-filled once and cut into, for every
layer call that owns a cache and every tensor its mixer caches, a view
[pages, *leading axes, page_size, last axis] (for attention: K and V
[pages, heads, page_size, head_dim], so that a (page, head) is one contiguous
[page_size, head_dim] box; for a tensor kept per page [pages, *axes]); and per
state-keeping layer call one pool [slots, *state shape]
(reference layout of the pages: src/cuda/model/kv_cache.cpp:17-52, src/cuda/kernels/kernels.h:15-27)."""

from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import torch

from ..parts.base import LayerCache
from ..parts.spec import CacheTensor, StateSpec
from .manager import GroupInfo


def bytes_per_page(groups: Sequence[GroupInfo], page_size: int, elem_size: int) -> List[int]:
    def of(t: CacheTensor) -> int:
        return t.page_elements(page_size) * (elem_size if t.dtype is None else getattr(torch, t.dtype).itemsize)
    return [len(g.owners) * sum(of(t) for t in g.spec.tensors) for g in groups]


ALIGN = 256        # bytes: where the tensors of a group that mixes types start


class CacheStorage:
    def __init__(self, groups: Sequence[GroupInfo], pages_per_group: Sequence[int], page_size: int,
                 dtype: torch.dtype, device: torch.device):
        self.page_size = page_size
        self.pools: List[torch.Tensor] = []
        self._by_owner: Dict[int, LayerCache] = {}
        for gi, (g, n) in enumerate(zip(groups, pages_per_group)):
            if g.spec.typed():
                self._add_typed(gi, g, n, dtype, device)
                continue
            per_owner = n * page_size * g.spec.elements_per_token()
            pool = torch.zeros(max(len(g.owners), 1) * per_owner, dtype=dtype, device=device)
            self.pools.append(pool)
            for j, owner in enumerate(g.owners):
                views: Dict[str, torch.Tensor] = {}
                off = j * per_owner
                for t in g.spec.tensors:
                    size = n * page_size * t.elements()
                    views[t.name] = pool[off:off + size].view((n,) + tuple(t.shape[:-1]) + (page_size, t.shape[-1]))
                    off += size
                self._by_owner[owner] = LayerCache(gi, views, True)

    def _add_typed(self, gi: int, g: GroupInfo, n: int, dtype: torch.dtype, device: torch.device) -> None:
        """A group whose tensors name their types: one allocation of bytes."""
        parts = []                  # (name, type, first byte, bytes, shape) within an owner's share
        per_owner = 0
        for t in g.spec.tensors:
            dt = dtype if t.dtype is None else getattr(torch, t.dtype)
            size = n * t.page_elements(self.page_size) * dt.itemsize
            parts.append((t.name, dt, per_owner, size, (n,) + t.page_shape(self.page_size)))
            per_owner += (size + ALIGN - 1) // ALIGN * ALIGN
        pool = torch.zeros(max(len(g.owners), 1) * per_owner, dtype=torch.uint8, device=device)
        self.pools.append(pool)
        for j, owner in enumerate(g.owners):
            first = j * per_owner
            self._by_owner[owner] = LayerCache(gi, {name: pool[first + at:first + at + size].view(dt).view(shape)
                                                    for name, dt, at, size, shape in parts}, True)

    def of_owner(self, owner: int, write: bool) -> LayerCache:
        c = self._by_owner[owner]
        return c if write else LayerCache(c.group, c.tensors, False)

    def nbytes(self) -> int:
        return sum(p.numel() * p.element_size() for p in self.pools)


class StateStorage:
    """Pools of fixed-size per-request state, one per layer call that keeps state.  A pool has one slot more
    than the manager hands out: index ``num_slots`` belongs to the padding rows of fixed-shape batches."""

    def __init__(self, specs: Dict[int, StateSpec], num_slots: int, device: torch.device):
        """``specs[call]`` is one ``StateSpec`` or a tuple of them (the call then gets a tuple of pools)."""
        def pool(s: StateSpec) -> torch.Tensor:
            return torch.zeros((num_slots + 1,) + tuple(s.shape), dtype=getattr(torch, s.dtype), device=device)

        self.pools: Dict[int, object] = {
            call: tuple(pool(x) for x in s) if isinstance(s, (tuple, list)) else pool(s) for call, s in specs.items()
        }

    def _all(self):
        for p in self.pools.values():
            yield from (p if isinstance(p, tuple) else (p,))

    def snapshot(self) -> List[torch.Tensor]:
        return [p.clone() for p in self._all()]

    def restore(self, saved: List[torch.Tensor]) -> None:
        for p, old in zip(self._all(), saved):
            p.copy_(old)

    def of_call(self, call: int):
        return self.pools.get(call)

    def reset_slot(self, slot: int) -> None:
        for p in self._all():
            p[slot].zero_()

    def nbytes(self) -> int:
        return sum(p.numel() * p.element_size() for p in self._all())
