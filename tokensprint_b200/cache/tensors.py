"""Device memory of the cache: page pools per cache, state slots per cache."""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from tokensprint_b200 import ops
from tokensprint_b200.cache.manager import GroupSpec
from tokensprint_b200.parts.base import CacheNeed, LayerCache


def groups_of(needs: Sequence[CacheNeed]) -> tuple[list[GroupSpec], list[int]]:
    """Sorts caches into groups by paging need.  Returns the groups and, for every cache,
    the index of its group (-1 for a cache without pages)."""
    keys: list[tuple[str, int]] = []
    index: list[int] = []
    for need in needs:
        if need.kind == "none":
            index.append(-1)
            continue
        if need.group_key not in keys:
            keys.append(need.group_key)
        index.append(keys.index(need.group_key))
    return [GroupSpec(kind, window) for kind, window in keys], index


def page_bytes(needs: Sequence[CacheNeed], group_index: Sequence[int], group: int, page_size: int, itemsize: int, kv4: bool = False,
               weighed: bool = False) -> int:
    """Bytes one page of `group` costs over all caches of the group (keys and values; `kv4`: in 4 bits; `weighed`: with a weight per row and head)."""
    if kv4:
        per_head = [(n.k_row[0], 9 * n.k_row[1] // 8 + (4 if weighed else 0)) for n, g in zip(needs, group_index) if g == group]
        return sum(page_size * heads * size for heads, size in per_head)
    return sum(page_size * n.token_elements * itemsize for n, g in zip(needs, group_index) if g == group)


@dataclass
class CacheTensors:
    """Per cache: the pools [pages, page_size, *k_row] and [pages, page_size, *v_row] (the second
    may be absent or of another row shape) and the state [slots, ...].  A cache in 4 bits has one pool instead
    (`kv4`, ops.kv4_pool_shape) and, where rows are weighed, their weights (`sums`, [pages, heads, page_size])."""

    k: list[Optional[torch.Tensor]]
    v: list[Optional[torch.Tensor]]
    state: list[Optional[torch.Tensor]]
    group_index: list[int]
    kv4: list[Optional[torch.Tensor]]
    sums: list[Optional[torch.Tensor]]

    @classmethod
    def allocate(
        cls,
        needs: Sequence[CacheNeed],
        group_index: Sequence[int],
        pages_per_group: Sequence[int],
        page_size: int,
        num_slots: int,
        device: torch.device,
        dtype: torch.dtype,
        kv4: bool = False,
        weighed: bool = False,
    ) -> "CacheTensors":
        k, v, state, pools, sums = [], [], [], [], []
        for need, g in zip(needs, group_index):
            packed = kv4 and g >= 0
            pools.append(torch.zeros(ops.kv4_pool_shape(pages_per_group[g], page_size, *need.k_row), device=device, dtype=torch.uint8) if packed else None)
            sums.append(torch.zeros((pages_per_group[g], need.k_row[0], page_size), device=device) if packed and weighed else None)
            if packed:
                k.append(None)
                v.append(None)
            elif g >= 0:
                k.append(torch.zeros((pages_per_group[g], page_size, *need.k_row), device=device, dtype=dtype))
                v.append(None if need.v_row is None else
                         torch.zeros((pages_per_group[g], page_size, *need.v_row), device=device, dtype=dtype))
            else:
                k.append(None)
                v.append(None)
            if need.state_shape is not None:
                state.append(torch.zeros((num_slots, *need.state_shape), device=device, dtype=need.state_dtype))
            else:
                state.append(None)
        return cls(k, v, state, list(group_index), pools, sums)

    def layer_cache(self, cache: int, writes: bool, read_later: int = 0) -> LayerCache:
        return LayerCache(
            group=self.group_index[cache],
            k_pages=self.k[cache],
            v_pages=self.v[cache],
            state=self.state[cache],
            writes=writes,
            read_later=read_later,
            kv4_pool=self.kv4[cache],
            kv4_sums=self.sums[cache],
        )

    def zero_slot(self, slot: int) -> None:
        for s in self.state:
            if s is not None:
                s[slot].zero_()

    def poison_pages(self, group: int, pages: Sequence[int]) -> None:
        """Debug aid: NaN (in a 4-bit cache, the largest scales) into pages that were given back, so a stale read shows."""
        if not pages:
            return
        idx = None
        for c, g in enumerate(self.group_index):
            if g == group and self.kv4[c] is not None:
                self.kv4[c][torch.tensor(list(pages), device=self.kv4[c].device, dtype=torch.long)] = 0xFF
            if g == group and self.k[c] is not None:
                if idx is None:
                    idx = torch.tensor(list(pages), device=self.k[c].device, dtype=torch.long)
                self.k[c][idx] = float("nan")
                if self.v[c] is not None:
                    self.v[c][idx] = float("nan")
