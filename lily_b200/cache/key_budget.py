"""Holding a paged cache to a budget of places: the keys that attention gave the least weight to are let go of.

Beside the pages of each cache group lie the weights of their places, float32 ``[layers, pages + 1, kv_heads, page_size]``:
what the queries so far gave each cached key (``ops.attention_key_weights`` for prompt portions,
``ops.attention_decode_weighed`` for decoded tokens add to them).  A request that has grown ``slack`` places past
``keep`` is brought back to ``keep``: every kv head of every layer keeps its own first ``first`` places, its last
``recent`` and the heaviest of the rest (``ops.select_keys``), moved to the front of the request's pages in their order
(``ops.move_keys``), and the pages behind go back to the pool.

From then on a token's place in the cache is not its position: keys were rotated by their positions when they were
written and stay so, the next token is written behind the kept places (``ops.axes_rope_write`` takes place and position apart), and the
caller counts positions.  ``slack`` spreads the cost: with 128 a request is evicted once in 128 decoded tokens.

A key that was let go of does not come back, so an eviction first waits for the work that the weights come from and looks whether a kernel of
it gave up a wait (``check_waits``): it raises then, and nothing has been let go of.

The reference keeps every key of a request until it ends (lily/mem_cache/memory_pool.py:78-143) or slides a window.
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np
import torch

from lily_b200.cache.kv_cache import KVCacheManager
from lily_b200.csrc.waits import Listener


class KeyBudget:
    def __init__(self, cache: KVCacheManager, keep: int, *, first: int = 4, recent: Optional[int] = None, slack: int = 128, ops=None):
        recent = keep // 4 if recent is None else recent
        if keep < 1 or first < 0 or recent < 0 or first + recent > keep or slack < 1:
            raise ValueError(f"a budget of {keep} places keeps the first {first} and the last {recent} of them, and lets {slack} come on top")
        if cache.device is None:
            raise ValueError("a cache without device tensors has nothing to evict")
        for g in cache.groups:
            if g.need.window is not None or g.need.values_in_keys or g.need.v_head_dim not in (None, g.need.head_dim):
                raise ValueError("a budget is for caches of all keys, with keys and values of one head size")
        if cache.state_needs:
            raise ValueError("a mixer with a state of its own does not live on cached keys alone")
        if ops is None:
            from lily_b200.csrc import ops
        self.cache, self.ops, self._waits = cache, ops, Listener(ops)
        self.keep, self.first, self.recent, self.slack = keep, first, recent, slack
        self.weights: List[torch.Tensor] = [
            torch.zeros((g.num_layers, cache.num_pages + 1, g.need.kv_heads, cache.page_size), dtype=torch.float32, device=cache.device) for g in cache.groups]

    def layer(self, group: int, index: int) -> torch.Tensor:
        """The weights of one layer, beside ``cache.groups[group].layer(index)``."""
        return self.weights[group][index]

    @property
    def most(self) -> int:
        """Places a request may hold between two evictions (what a decode step plans for)."""
        return self.keep + self.slack

    def table(self, group: int, slots: Sequence[int], width: int = 0) -> torch.Tensor:
        """The block tables of these requests, int32 [requests, pages] on the device (0 behind the last page)."""
        rows = [self.cache.block_table(group, s) for s in slots]
        host = np.zeros((len(rows), max([width, 1] + [len(r) for r in rows])), dtype=np.int32)
        for i, r in enumerate(rows):
            host[i, :len(r)] = r
        return torch.from_numpy(host).to(self.cache.device, non_blocking=True)

    def check_waits(self, wait: bool = False) -> None:
        """Raises when a kernel that weighs keys gave up a wait of its own, so that what came of its step is void: in the work that the host has waited
        for, or (``wait``) in all that is enqueued on the current stream."""
        if wait and torch.device(self.cache.device).type == "cuda":
            torch.cuda.current_stream(self.cache.device).synchronize()
        self._waits.check()

    def evict(self, slots: Sequence[int], force: bool = False) -> List[int]:
        """Brings those of these requests that hold ``slack`` places or more past the budget (with ``force``: any past it) back to it and
        gives their slots.  Where there are some, the host first waits for the current stream and looks for waits that ran out
        (``check_waits``); the rest is enqueued, and the pages behind are free for what is enqueued after."""
        over = [s for s in dict.fromkeys(slots) if self.cache.lengths[s] >= self.keep + (1 if force else self.slack)]
        if not over:                       # (a request that is named twice is moved once: two moves in place would meet)
            return []
        held = [self.cache.lengths[s] for s in over]
        lengths = torch.tensor(held, dtype=torch.int32).to(self.cache.device, non_blocking=True)
        tables = [self.table(g, over) for g in range(len(self.cache.groups))]
        self.check_waits(wait=True)
        for g, (group, table) in enumerate(zip(self.cache.groups, tables)):
            kept = self.ops.select_keys(self.weights[g], table, lengths, max(held), self.keep, self.first, self.recent)
            self.ops.move_keys(group.data, self.weights[g], table, kept)
        for s in over:
            self.cache.shrink(s, self.keep)
        return over


__all__ = ["KeyBudget"]
