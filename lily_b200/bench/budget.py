"""A stack of attention layers whose cache is held to a budget, beside the same stack with every key kept.

    python -m lily_b200.bench.budget                                  (Qwen3-8B attention sizes, 8 layers, 8 requests)
    python -m lily_b200.bench.budget --prompt 16384 --keep 2048 --image

Every request brings a prompt (``--image``: half of it an image, whose tokens have a time, a row and a column), in portions, then decodes
one token a step.  With the budget the keys that attention gave the least weight to are let go of behind every portion and
every ``slack`` decoded tokens (``lily_b200.cache.key_budget``), so a decode step reads ``keep`` to ``keep + slack`` places of
each request however long it is.  Weights are random; what is printed is time and memory.

``AttentionStack`` is the whole path through the public entry points: product, norm + rotation + cache write
(``axes_rope_write``), attention (``attention_prefill`` with ``attention_key_weights``, or ``attention_decode_weighed``), output
product, eviction.
"""

from __future__ import annotations

import argparse
import json
import math
from typing import List, Optional, Sequence

import torch

from lily_b200.cache.key_budget import KeyBudget
from lily_b200.cache.kv_cache import KVCacheManager
from lily_b200.csrc.waits import Listener
from lily_b200.parts.base import CacheNeed


def image_prompt(text: int, rows: int, columns: int, behind: int, start: int = 0) -> torch.Tensor:
    """Positions [3, tokens] (time, row, column) of ``text`` tokens, an image of rows x columns patches, and ``behind`` tokens: text
    moves along all axes alike, the patches stand at one time, and what follows goes on behind the largest of them."""
    i = torch.arange(rows * columns)
    at = start + text
    patches = at + torch.stack([torch.zeros_like(i), i // max(1, columns), i % max(1, columns)])
    last = at + max(1 if rows * columns else 0, rows, columns)
    line = lambda first, n: (first + torch.arange(n)).expand(3, n)
    return torch.cat([line(start, text), patches, line(last, behind)], 1).to(torch.int32)


class AttentionStack:
    """``layers`` of x <- x + W_o attention(W_qkv x): grouped heads with per-head norm, positions with three axes, one paged cache."""

    def __init__(self, layers: int, width: int, nq: int, nkv: int, d: int, *, page_size: int = 64, num_pages: int, max_requests: int, max_context: int,
                 max_position: int, device="cuda", dtype=torch.bfloat16, seed: int = 0, ops=None, keep: Optional[int] = None, first: int = 4,
                 recent: Optional[int] = None, slack: int = 128, sections: Optional[Sequence[int]] = None):
        if ops is None:
            from lily_b200.csrc import ops
        self.ops, self.device, self.dtype = ops, torch.device(device), dtype
        self.layers, self.nq, self.nkv, self.d, self.page = layers, nq, nkv, d, page_size
        self.cache = KVCacheManager([(CacheNeed(nkv, d), layers)], [], page_size=page_size, num_pages=num_pages, max_requests=max_requests,
                                    max_context=max_context, dtype=dtype, device=self.device)
        self.budget = KeyBudget(self.cache, keep, first=first, recent=recent, slack=slack, ops=ops) if keep else None
        g = torch.Generator().manual_seed(seed)
        row = (nq + 2 * nkv) * d
        draw = lambda *shape: (torch.randn(*shape, generator=g) / math.sqrt(shape[-1])).to(dtype).to(self.device)
        self.w_qkv = [draw(row, width) for _ in range(layers)]
        self.w_o = [draw(width, nq * d) for _ in range(layers)]
        self.gain = [(1 + 0.1 * torch.randn(d, generator=g)).to(dtype).to(self.device) for _ in range(2)]
        half = d // 2
        sections = sections or (half // 4, (half - half // 4) // 2, half - half // 4 - (half - half // 4) // 2)
        self.pair_axis = ops.pair_axes(sections, self.device)
        angle = torch.outer(torch.arange(max_position, dtype=torch.float32), 1.0 / 10000.0 ** (torch.arange(0, d, 2, dtype=torch.float32) / d))
        self.cos, self.sin = angle.cos().to(self.device), angle.sin().to(self.device)
        self.check_waits = self.budget.check_waits if keep else Listener(ops).check        # raises when an attention kernel of a step that the host has waited for gave up a wait
        self.next_position = {}                       # by slot: the caller of a budgeted cache counts positions

    # ---- requests --------------------------------------------------------------------

    def open(self) -> int:
        slot = self.cache.open_request()
        self.next_position[slot] = 0
        return slot

    def close(self, slot: int) -> None:
        self.cache.close_request(slot)
        del self.next_position[slot]

    # ---- steps -----------------------------------------------------------------------

    def _dev(self, values, dtype=torch.int32) -> torch.Tensor:
        return torch.as_tensor(values, dtype=dtype).to(self.device, non_blocking=True)

    def _table(self, slots: Sequence[int]) -> torch.Tensor:
        if self.budget is not None:
            return self.budget.table(0, slots)
        rows = [self.cache.block_table(0, s) for s in slots]
        width = max(1, max(len(r) for r in rows))
        return self._dev([r + [0] * (width - len(r)) for r in rows])

    def _heads(self, layer: int, x, positions, places, req, table):
        return self.ops.axes_rope_write(self.ops.linear_auto(x.to(self.dtype), self.w_qkv[layer]), *self.gain, 1e-6, self.cos, self.sin, positions, self.pair_axis, places,
                                        req, table, self.cache.groups[0].layer(layer), self.nq, self.nkv, self.d, self.d, self.page)

    def _close_layer(self, layer: int, x, out):
        return x + self.ops.linear(out, self.w_o[layer]).to(x.dtype)

    def portion(self, slots: Sequence[int], xs: Sequence[torch.Tensor], positions: Sequence[torch.Tensor], observe: Optional[int] = None) -> List[torch.Tensor]:
        """The next portion of several requests' prompts: rows ``xs[i]`` [n, width] at ``positions[i]`` [3, n].  Returns what the stack makes of
        them; the last ``observe`` tokens of each portion (all by default) say which keys are heavy."""
        new = [x.shape[0] for x in xs]
        cached = [self.cache.lengths[s] for s in slots]
        for s, p, n in zip(slots, cached, new):
            self.cache.grow(s, p + n)
        for s, at in zip(slots, positions):
            self.next_position[s] = int(at.max()) + 1
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        table, cu_dev, prefix = self._table(slots), self._dev(cu), self._dev(cached)
        at = torch.cat([p.to(torch.int32) for p in positions], 1).contiguous().to(self.device)
        places = self._dev([p + t for p, n in zip(cached, new) for t in range(n)])
        req = self._dev([i for i, n in enumerate(new) for _ in range(n)])
        rows = self.ops.prefill_tile_rows(self.dtype, self.d, self.page, cu[-1])
        tile_req, tile_start = self.ops.prefill_tiles(cached, new, 0, rows, self.device)
        x = torch.cat(list(xs)).float()
        for layer in range(self.layers):
            kv, scale = self.cache.groups[0].layer(layer), self.d ** -0.5
            q = self._heads(layer, x, at, places, req, table)
            out = torch.empty_like(q)
            self.ops.attention_prefill(q, kv, table, cu_dev, prefix, tile_req, tile_start, out, self.nq, self.nkv, self.d, self.page, scale, tile_rows=rows)
            if self.budget is not None:
                self.ops.attention_key_weights(q, kv, self.budget.layer(0, layer), table, cu_dev, prefix, cached, new, self.nq, self.nkv, self.d, self.page, scale,
                                               observe=observe)
            x = self._close_layer(layer, x, out)
        if self.budget is not None:
            self.budget.evict(slots)
        return list(x.split(new))

    def decode(self, slots: Sequence[int], x: torch.Tensor) -> torch.Tensor:
        """One token of every request: rows of ``x`` [requests, width]."""
        n = len(slots)
        cached = [self.cache.lengths[s] for s in slots]
        for s, p in zip(slots, cached):
            self.cache.grow(s, p + 1)
        longest = max(cached) + 1
        table, places, seq = self._table(slots), self._dev(cached), self._dev([p + 1 for p in cached])
        at, req = self._dev([[self.next_position[s] for s in slots]] * 3), self._dev(list(range(n)))
        for s in slots:
            self.next_position[s] += 1
        x = x.float()
        for layer in range(self.layers):
            kv, scale = self.cache.groups[0].layer(layer), self.d ** -0.5
            q = self._heads(layer, x, at, places, req, table)
            if self.budget is not None:
                out = self.ops.attention_decode_weighed(q, kv, self.budget.layer(0, layer), table, seq, longest, self.nq, self.nkv, self.d, self.page, scale)
            else:
                plan = self.ops.plan_decode_attention(self.dtype, n, self.nq, self.nkv, self.d, longest, fusable=False)
                out = torch.empty_like(q)
                scratch = torch.empty(max(1, plan.scratch_floats), device=self.device)
                self.ops.attention_decode(q, kv, table, seq, out, scratch, plan.splits, self.nq, self.nkv, self.d, self.page, scale, stages=plan.stages)
            x = self._close_layer(layer, x, out)
        if self.budget is not None:
            self.budget.evict(slots)
        return x


def measure(args, keep: Optional[int]) -> dict:
    most = args.prompt + args.steps + 64
    room = min(most, (keep or most) + args.slack + args.portion) + args.page
    stack = AttentionStack(args.layers, args.width, args.heads, args.kv_heads, args.head_dim, page_size=args.page, num_pages=args.rows * -(-room // args.page) + 1,
                           max_requests=args.rows, max_context=most, max_position=most, keep=keep, slack=args.slack)
    slots = [stack.open() for _ in range(args.rows)]
    g = torch.Generator(device="cuda").manual_seed(1)
    side = math.isqrt(args.prompt // 2) if args.image else 0
    text = (args.prompt - side * side) // 2
    where = image_prompt(text, side, side, args.prompt - side * side - text)

    def timed(step):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        step()
        end.record()
        torch.cuda.synchronize()
        return start.elapsed_time(end)

    def prompts():
        for p in range(0, args.prompt, args.portion):
            n = min(args.portion, args.prompt - p)
            stack.portion(slots, [torch.randn(n, args.width, device="cuda", generator=g) for _ in slots], [where[:, p:p + n] for _ in slots])
    fill = timed(prompts)
    if stack.budget is not None:
        stack.budget.evict(slots, force=True)
    row = torch.randn(args.rows, args.width, device="cuda", generator=g)
    times = sorted(timed(lambda: stack.decode(slots, row)) for _ in range(args.steps))
    stack.check_waits()
    data = stack.cache.groups[0].data
    return {"keep": keep, "prompt_ms": round(fill, 2), "decode_ms_median": round(times[len(times) // 2], 3), "decode_ms_worst": round(times[-1], 3),
            "places": stack.cache.lengths[slots[0]], "cache_mb": round(data.numel() * data.element_size() / 2 ** 20, 1)}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("layers", 8), ("width", 4096), ("heads", 32), ("kv-heads", 8), ("head-dim", 128), ("page", 64), ("rows", 8), ("prompt", 8192), ("portion", 2048),
                          ("keep", 1024), ("slack", 128), ("steps", 160)):
        ap.add_argument("--" + name, type=int, default=default)
    ap.add_argument("--image", action="store_true")
    args = ap.parse_args()
    for keep in (None, args.keep):
        measure(argparse.Namespace(**{**vars(args), "prompt": min(args.prompt, args.portion), "steps": 4}), keep)        # libraries and kernels set themselves up
        print(json.dumps(measure(args, keep)))


if __name__ == "__main__":
    main()
