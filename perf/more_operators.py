"""What the operators of serving in four bits are measured on.

Weights and the key/value cache are held in four bits and everything else stays as it is: activations, norms, rotation, softmax and sums are
those of the bfloat16 (or float32) engine.  Four kinds of case:

* ``product``   x W^T with W in 4-bit codes, a scale (and perhaps a zero point) for each group of a row's columns: one token, a few, a
                server's worth of users, a prompt.
* ``write``     per-head norm, rotation, queries out, keys and values into a 4-bit paged cache; then the values the touched pages stand for.
* ``decode``    attention of one new token a request over its 4-bit pages.
* ``portions``  causal attention of prompt portions (``n@p``: n new tokens behind p cached ones), whose keys are in the 4-bit pages already.

How numbers are held.  Weights: ``codes`` uint8 [ceil(n / 128), ceil(k / 128), 128, 64], rows and columns in tiles of 128; a row of a tile
is 16 words of 8 codes (the lowest bits first), word 4 t + w holding columns 32 w + 8 t + (0..7); ``scales`` bfloat16 [ceil(n / 128),
groups, 128] and ``zeros`` uint8 of that shape or none (then 8): W = scale (code - zero).  Cache: uint8 [pages, kv_heads, 2 (keys,
values), page_size (d / 2 + d / 16)]: the places' codes, then for each place and group of 64 features two bfloat16 numbers, step and lowest
value: x = lowest + step code.  A place's codes are words of 8 again: word 8 j + 4 h + t of a key (j the group) lies at (t, j, h),
word 8 j + g of a value at (g, j).

Sizes are those of ``perf/cases.py``: "small" (width 2,048, 16 query heads over 4 kv heads of 128) and "mid" (4,096, 32 over 8, 12,288).
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
TABLE = 32768                    # positions in the rotation tables
GROUP = 64                       # features of a head that share a step and a lowest value in the cache


def listed():
    return [
        # one user of a small model, its output projection: the smallest call
        {"name": "product-1", "kind": "product", "dtype": "bf16", "tokens": 1, "n": 2048, "k": 2048, "group": 128, "zeros": False},
        # the gate/up product of a decode step of eight users
        {"name": "product-8", "kind": "product", "dtype": "bf16", "tokens": 8, "n": 24576, "k": 4096, "group": 128, "zeros": False},
        # the down product of a busier server, finer groups with zero points, as calibrated checkpoints have them
        {"name": "product-45", "kind": "product", "dtype": "bf16", "tokens": 45, "n": 4096, "k": 12288, "group": 64, "zeros": True},
        # a prompt through the stacked q, k, v projection
        {"name": "product-2048", "kind": "product", "dtype": "bf16", "tokens": 2048, "n": 6144, "k": 4096, "group": 128, "zeros": False},
        # checking a checkpoint in 32-bit, odd rows
        {"name": "product-f32", "kind": "product", "dtype": "f32", "tokens": 3, "n": 2049, "k": 8192, "group": 32, "zeros": True},
        # a decode step of eight users: one row each into the cache
        {"name": "write-8", "kind": "write", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "rot": 128, "page": 64, "tokens": "1,1,1,1,1,1,1,1", "norm": True},
        # ragged prompts
        {"name": "write-1500", "kind": "write", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "rot": 128, "page": 64, "tokens": "1103,1,396", "norm": True},
        # eight users with long contexts
        {"name": "decode-8", "kind": "decode", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "page": 64, "rows": 8, "low": 8192, "high": 8192, "empty": False},
        # a busy server: 64 users with contexts of very different lengths
        {"name": "decode-64", "kind": "decode", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "page": 64, "rows": 64, "low": 250, "high": 1750, "empty": False},
        # checking a checkpoint in 32-bit; a slot of the step without a request
        {"name": "decode-f32", "kind": "decode", "dtype": "f32", "nq": 16, "nkv": 4, "d": 128, "page": 16, "rows": 3, "low": 150, "high": 2900, "empty": True},
        # one prompt
        {"name": "portions-2048", "kind": "portions", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "page": 64, "portions": "2048"},
        # a later portion of a long prompt beside a short prompt and the last token of one
        {"name": "portions-mixed", "kind": "portions", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "page": 64, "portions": "600@5000,333,1@511"},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["product", "product", "write", "decode", "portions"])
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    if kind == "product":
        group = rng.choice([32, 64, 128, 128])
        n, k = _log(rng, 64, 26000), group * _log(rng, 128 // group, 12800 // group)
        few = rng.random() < 0.6
        tokens = _log(rng, 1, 16) if few else _log(rng, 17, 2048 if dtype == "bf16" else 200)
        most = 5e10 if dtype == "bf16" else 6e9
        return {"kind": kind, "dtype": dtype, "tokens": max(1, min(tokens, int(most / (n * k)))), "n": n, "k": k, "group": group, "zeros": rng.random() < 0.4}
    nq, nkv, d = rng.choice([(16, 4, 128), (32, 8, 128), (16, 16, 64), (12, 4, 64), (14, 2, 64), (24, 2, 128), (8, 4, 256)])
    c = {"kind": kind, "dtype": dtype, "nq": nq, "nkv": nkv, "d": d, "page": rng.choice([16, 64, 64, 128])}
    if kind == "write":
        rows = rng.random() < 0.4
        c["tokens"] = ",".join(["1"] * _log(rng, 1, 64)) if rows else ",".join(str(_log(rng, 2, 500)) for _ in range(rng.randint(1, 3)))
        c.update(rot=d if rng.random() < 0.7 else d // 2, norm=rng.random() < 0.6)
    elif kind == "decode":
        c["rows"] = _log(rng, 1, 64)
        c["high"] = _log(rng, 1, min(32768, 60000 // c["rows"]) // (4 if dtype == "f32" else 1))
        c["low"] = _log(rng, max(1, c["high"] // 8), c["high"])
        c["empty"] = rng.random() < 0.2
    else:
        top = 500 if dtype == "f32" else 1100
        c["portions"] = ",".join(f"{_log(rng, 1, top)}@{rng.choice([0, _log(rng, 1, 2 * top)])}" for _ in range(rng.randint(1, 3)))
    return c


def _lengths(case):
    """``rows`` lengths spread between ``low`` and ``high`` (both among them); the middle one is nothing where a slot is ``empty``."""
    n, low, high = case["rows"], case["low"], case["high"]
    lengths = [high] if n == 1 else [round(low * (high / low) ** ((i * 5 % n if n % 5 else i) / (n - 1))) for i in range(n)]
    if case["empty"] and n > 1:
        lengths[n // 2] = 0
    return lengths


def _portions(case):
    """(new, cached) of every portion."""
    return [tuple(int(x) for x in (p.split("@") + ["0"])[:2]) for p in case["portions"].split(",")]


def work(case):
    item = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "product":
        m, n, k, groups = case["tokens"], case["n"], case["k"], case["k"] // case["group"]
        return {"bytes": n * k // 2 + n * groups * (3 if case["zeros"] else 2) + m * (n + k) * item, "flops": 2 * m * n * k}
    d, nq, nkv = case["d"], case["nq"], case["nkv"]
    held = d // 2 + d // 16
    if case["kind"] == "write":
        tokens = [int(x) for x in case["tokens"].split(",")]
        n, page = sum(tokens), case["page"]
        places = sum(-(-(c + t) // page) * page for c, t in zip(_cached(case, tokens), tokens))
        return {"bytes": n * ((2 * nq + 2 * nkv) * d * item + 4 * case["rot"] + 2 * nkv * held) + places * 2 * nkv * (held + d * item), "flops": n * (nq + 2 * nkv) * d * 8}
    if case["kind"] == "decode":
        places = sum(_lengths(case))
        return {"bytes": places * nkv * 2 * held + case["rows"] * nq * d * 2 * item, "flops": 4 * places * nq * d}
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in _portions(case))
    return {"bytes": sum((n + p) * nkv * 2 * held + 2 * n * nq * d * item for n, p in _portions(case)), "flops": 4 * pairs * nq * d}


# ------------------------------------------------------------------------------ what a program has in hand

def _cached(case, tokens):
    return [(37 * i + 5) % (3 * case["page"]) for i in range(len(tokens))]


def _pages(lengths, page, g):
    """Block tables over shuffled pages, and the pages of the pool (page 0 belongs to nobody)."""
    counts = [-(-n // page) for n in lengths]
    total = sum(counts) + 3
    order = torch.randperm(total, generator=g)[:sum(counts)] + 1
    table = torch.nn.utils.rnn.pad_sequence(order.split(counts), batch_first=True)
    table = torch.nn.functional.pad(table, (0, max(0, 1 - table.shape[1])))
    return table.int().contiguous().to(DEV), total


def _nibbles(codes):
    """The two codes of every byte, the lower one first, along the last axis."""
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _bytes(codes):
    pairs = codes.unflatten(-1, (-1, 2))
    return pairs[..., 0] | (pairs[..., 1] << 4)


def _tiled(x, fill):
    """Rows and columns of ``x`` [n, k] in tiles of 128 [n / 128, k / 128, 128, 128], filled up."""
    n, k = x.shape
    return torch.nn.functional.pad(x, (0, -k % 128, 0, -n % 128), value=fill).unflatten(1, (-1, 128)).unflatten(0, (-1, 128)).transpose(1, 2)


def _hold(x):
    """Heads [..., d] as (codes 0..15 uint8 [..., d], step and lowest bfloat16 [..., d / 64, 2]); a group that is not finite has neither."""
    x = x.unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    step, low = ((high - low) * (1.0 / 15.0)).bfloat16(), low.bfloat16()
    bad = ~(torch.isfinite(step) & torch.isfinite(low))
    step, low = step.masked_fill(bad, math.nan), low.masked_fill(bad, math.nan)
    code = torch.round((x - low.float()[..., None]) / step.float()[..., None]).clamp(0, 15)
    code = torch.where((step > 0)[..., None], code, 0.0).to(torch.uint8)
    return code.flatten(-2), torch.stack([step, low], -1)


def _key_bytes(codes):
    """Codes [..., d] of keys as bytes [..., d / 2] in their order; of values, below."""
    groups = codes.shape[-1] // GROUP
    return _bytes(codes.unflatten(-1, (groups, 2, 4, 8)).movedim(-2, -4)).flatten(-4)


def _value_bytes(codes):
    groups = codes.shape[-1] // GROUP
    return _bytes(codes.unflatten(-1, (groups, 8, 8)).transpose(-3, -2)).flatten(-3)


def _parts(kv, page, d):
    """(codes [..., page, d / 2], steps and lowest values [..., page, d / 64, 2]) of cache rows [..., page (d / 2 + d / 16)], as views."""
    return kv[..., :page * d // 2].unflatten(-1, (page, d // 2)), kv[..., page * d // 2:].view(torch.bfloat16).unflatten(-1, (page, d // GROUP, 2))


def _values(rows, page, d, of_values):
    """What cache rows [..., page (d / 2 + d / 16)] stand for, float32 [..., page, d]."""
    codes, held = _parts(rows, page, d)
    groups = d // GROUP
    if of_values:
        c = _nibbles(codes.unflatten(-1, (8, groups, 4))).transpose(-3, -2)
    else:
        c = _nibbles(codes.unflatten(-1, (4, groups, 2, 4))).movedim(-4, -2)
    c = c.flatten(-3 if of_values else -4).unflatten(-1, (groups, GROUP)).float()
    held = held.float()
    return (held[..., 1:] + held[..., :1] * c).flatten(-2)


def prepare(case, seed):
    h = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, device=DEV, generator=g)
    s = {"case": case, "dtype": dtype}
    if case["kind"] == "product":
        n, k, groups = case["n"], case["k"], case["k"] // case["group"]
        loud = torch.where(torch.rand(k, device=DEV, generator=g) < 0.01, 8.0, 1.0)           # a few features are much larger than the others
        s["x"] = (randn(case["tokens"], k) * loud).to(dtype)
        codes = randn(n, k).mul_(2.6).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)
        s["codes"] = _bytes(_tiled(codes, 0).unflatten(-1, (4, 4, 8)).transpose(-3, -2)).flatten(-3).contiguous()
        held = lambda x: torch.nn.functional.pad(x, (0, -k % 128 // case["group"], 0, -n % 128)).unflatten(0, (-1, 128)).transpose(1, 2).contiguous()
        s["scales"] = held((randn(n, groups) * 0.3).exp() * (0.4 / math.sqrt(k))).bfloat16()
        s["zeros"] = held(torch.randint(5, 11, (n, groups), device=DEV, generator=g, dtype=torch.uint8)) if case["zeros"] else None
        return s
    nkv, d, page, nq = case["nkv"], case["d"], case["page"], case["nq"]
    if case["kind"] == "write":
        tokens = [int(x) for x in case["tokens"].split(",")]
        n, rot, cached = sum(tokens), case["rot"], _cached(case, tokens)
        s["table"], pages = _pages([c + t for c, t in zip(cached, tokens)], page, h)
        s["qkv"] = randn(n, (nq + 2 * nkv) * d).to(dtype)
        s["gains"] = [(1 + 0.2 * randn(d)).to(dtype) for _ in range(2)] if case["norm"] else [None, None]
        inv = 1.0 / 10000.0 ** (torch.arange(0, rot, 2, dtype=torch.float32) / rot)
        angle = torch.outer(torch.arange(TABLE, dtype=torch.float32), inv)
        s["cos"], s["sin"] = angle.cos().to(DEV), angle.sin().to(DEV)
        s["positions"] = torch.cat([c + torch.arange(t) for c, t in zip(cached, tokens)]).int().to(DEV)
        s["req"] = torch.repeat_interleave(torch.arange(len(tokens)), torch.tensor(tokens)).int().to(DEV)
        s["kv"] = _cache(randn(pages + 1, nkv, 2, page, d), page, d)
        return s
    if case["kind"] == "decode":
        lengths = _lengths(case)
        new = [1] * len(lengths)
        s["seq_lens"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        s["longest"] = max(lengths)
    else:
        new, cached = (list(x) for x in zip(*_portions(case)))
        lengths = [a + b for a, b in zip(new, cached)]
        s["new"], s["cached"] = new, cached
        s["prefix"] = torch.tensor(cached, dtype=torch.int32, device=DEV)
        s["cu"] = torch.tensor([0] + new).cumsum(0).int().to(DEV)
    s["table"], pages = _pages(lengths, page, h)
    lean = randn(nkv, d) / math.sqrt(d)
    kv = randn(pages + 1, nkv, 2, page, d)
    kv[:, :, 0] += (randn(pages + 1, nkv, page).exp() * 1.5)[..., None] * lean[:, None]        # some keys lean the queries' way
    s["kv"] = _cache(kv, page, d)
    s["q"] = (randn(sum(new), nkv, nq // nkv, d) + 3 * lean[:, None]).reshape(sum(new), nq * d).to(dtype)
    return s


def _cache(x, page, d):
    """Keys and values [pages, nkv, 2, page, d] as a 4-bit cache."""
    codes, held = _hold(x)
    codes = torch.stack([_key_bytes(codes[:, :, 0]), _value_bytes(codes[:, :, 1])], 2).flatten(-2)
    return torch.cat([codes, held.flatten(-3).view(torch.uint8)], -1).contiguous()


# ------------------------------------------------------------------------------ one pass

def run(s):
    return (_own if own else _plain)[s["case"]["kind"]](s)


def _own_product(s):
    from lily_b200.csrc import ops
    c = s["case"]
    return ops.linear4(s["x"], ops.Weight4(s["codes"], s["scales"], s["zeros"], c["n"], c["k"], c["group"]))


def _own_write(s):
    from lily_b200.csrc import ops
    c = s["case"]
    q = ops.qk_norm_rope_write4(s["qkv"], *s["gains"], EPS, s["cos"], s["sin"], s["positions"], s["req"], s["table"], s["kv"], c["nq"], c["nkv"], c["d"],
                                c["rot"], c["page"])
    return {"q": q, "values": ops.cache4_values(s["kv"], s["table"], c["nkv"], c["d"], c["page"], s["dtype"])}


def _own_decode(s):
    from lily_b200.csrc import ops
    c = s["case"]
    return ops.attention_decode4(s["q"], s["kv"], s["table"], s["seq_lens"], s["longest"], c["nq"], c["nkv"], c["d"], c["page"], c["d"] ** -0.5)


def _own_portions(s):
    from lily_b200.csrc import ops
    c = s["case"]
    return ops.attention_prefill4(s["q"], s["kv"], s["table"], s["cu"], s["prefix"], s["cached"], s["new"], c["nq"], c["nkv"], c["d"], c["page"], c["d"] ** -0.5)


def _plain_product(s):
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]
    codes = _nibbles(s["codes"].unflatten(-1, (4, 4, 4))).transpose(-3, -2).flatten(-3)          # [n tiles, k tiles, 128, 128]
    w = codes.transpose(1, 2).flatten(0, 1).flatten(1).float().unflatten(1, (-1, group))         # [rows, groups, group]
    rows = lambda t: t.transpose(1, 2).flatten(0, 1).float()[..., None]
    w = (rows(s["scales"]) * (w - (8.0 if s["zeros"] is None else rows(s["zeros"])))).flatten(1)
    return (s["x"].float() @ w[:n, :k].t()).to(s["dtype"])


def _turn(x, gain, cos, sin, rot):
    """Norm of the last axis where there is a gain, then rotation of its first ``rot`` features by halves."""
    if gain is not None:
        x = x * (1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)).float() * gain.float()
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def _plain_write(s):
    c = s["case"]
    nq, nkv, d, page, rot = c["nq"], c["nkv"], c["d"], c["page"], c["rot"]
    x = s["qkv"].float().view(-1, nq + 2 * nkv, d)
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q = _turn(x[:, :nq], s["gains"][0], cos, sin, rot).reshape(-1, nq * d).to(s["dtype"])
    pages, off = s["table"].long()[s["req"].long(), at // page], at % page
    codes, held = _parts(s["kv"], page, d)
    key, key_held = _hold(_turn(x[:, nq:nq + nkv], s["gains"][1], cos, sin, rot))
    value, value_held = _hold(x[:, nq + nkv:])
    codes[pages, :, 0, off], held[pages, :, 0, off] = _key_bytes(key), key_held
    codes[pages, :, 1, off], held[pages, :, 1, off] = _value_bytes(value), value_held
    kv = s["kv"][s["table"].long()]                                                                # [requests, pages, nkv, 2, ...]
    values = torch.stack([_values(kv[..., 0, :], page, d, False), _values(kv[..., 1, :], page, d, True)], 2)
    return {"q": q, "values": values.to(s["dtype"])}


def _gather(s, longest):
    """Keys and values of the places [0, longest) of every request, float32 [requests, nkv, longest, d]."""
    c = s["case"]
    kv = s["kv"][s["table"].long()].transpose(1, 2)                                                # [requests, nkv, pages, 2, ...]
    both = [_values(kv[..., i, :], c["page"], c["d"], bool(i)).flatten(2, 3)[:, :, :longest] for i in range(2)]
    return both[0], both[1]


def _plain_decode(s):
    c = s["case"]
    nq, nkv, d = c["nq"], c["nkv"], c["d"]
    k, v = _gather(s, s["longest"])
    lengths = s["seq_lens"].long()[:, None, None, None]
    q = s["q"].float().view(-1, nkv, nq // nkv, d)
    scores = (q @ k.transpose(-1, -2)) * d ** -0.5
    p = torch.softmax(scores.masked_fill(torch.arange(s["longest"], device=DEV) >= lengths, -math.inf), -1)
    return (p @ v).masked_fill(lengths == 0, 0.0).reshape(-1, nq * d).to(s["dtype"])


def _plain_portions(s):
    c = s["case"]
    nq, nkv, d = c["nq"], c["nkv"], c["d"]
    most = max(s["new"])
    longest = max(a + b for a, b in zip(s["new"], s["cached"]))
    k, v = _gather(s, longest)
    i, j = torch.arange(most, device=DEV), torch.arange(longest, device=DEV)
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    real = i < new[:, None]                                                                        # [requests, most]
    rows = torch.where(real, s["cu"][:-1].long()[:, None] + i, 0)
    q = s["q"].float()[rows].view(-1, most, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4)
    seen = j <= (s["prefix"].long()[:, None] + i)[..., None]                                       # [requests, most, longest]
    scores = (q @ k[:, :, None].transpose(-1, -2)).mul_(d ** -0.5).masked_fill_(~seen[:, None, None], -math.inf)
    out = torch.softmax(scores, -1) @ v[:, :, None]
    return out.permute(0, 3, 1, 2, 4)[real].reshape(-1, nq * d).to(s["dtype"])


_own = {"product": _own_product, "write": _own_write, "decode": _own_decode, "portions": _own_portions}
_plain = {"product": _plain_product, "write": _plain_write, "decode": _plain_decode, "portions": _plain_portions}


# ------------------------------------------------------------------------------ from the definitions, in 64 bits

def _places(row, page, d, value):
    """A cache row [.., page (d / 2 + d / 16)] of one page, kv head and kind as numbers in 64 bits, code by code from its place in the order."""
    codes = row[..., :page * d // 2].reshape(*row.shape[:-1], page, d // 2)
    held = row[..., page * d // 2:].contiguous().view(torch.bfloat16).double().reshape(*row.shape[:-1], page, d // GROUP, 2)
    f = torch.arange(d, device=DEV)
    j, word, i = f // GROUP, f % GROUP // 8, f % 8
    at = 4 * (word * (d // GROUP) + j if value else (word % 4) * 2 * (d // GROUP) + 2 * j + word // 4) + i // 2
    code = (codes[..., at] >> (4 * (i % 2)).to(torch.uint8)) & 15
    return held[..., j, 1] + held[..., j, 0] * code.double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "product":
        n, k, x = case["n"], case["k"], s["x"].double()
        f = torch.arange(k, device=DEV)
        within = f % 128
        at = 4 * (4 * (within % 32 // 8) + within // 32) + within % 8 // 2
        out = torch.empty(len(x), n, dtype=torch.float64, device=DEV)
        for r0 in range(0, n, 128):
            tile, rows = r0 // 128, min(128, n - r0)
            code = (s["codes"][tile, f // 128, :, at] >> (4 * (f % 2)).to(torch.uint8)[:, None]) & 15                  # [k, 128]
            zero = 8.0 if s["zeros"] is None else s["zeros"][tile, f // case["group"]].double()
            out[:, r0:r0 + rows] = (x @ ((code.double() - zero) * s["scales"][tile, f // case["group"]].double()))[:, :rows]
        return out
    nq, nkv, d, page = case["nq"], case["nkv"], case["d"], case["page"]
    if case["kind"] == "write":
        rot = case["rot"]
        heads = s["qkv"].double().view(-1, nq + 2 * nkv, d)
        phase = torch.complex(s["cos"][s["positions"].long()].double(), s["sin"][s["positions"].long()].double())[:, None]
        x = heads[:, :nq]
        if s["gains"][0] is not None:
            x = x / ((x * x).sum(-1, keepdim=True) / d + EPS).sqrt() * s["gains"][0].double()
        z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * phase
        # (which of two codes a number next to a border has is no matter of precision: the values have no counterpart in 64 bits)
        return {"q": torch.cat([z.real, z.imag, x[..., rot:]], -1).reshape(-1, nq * d), "values": None}
    group = nq // nkv
    q = s["q"].double().view(-1, nq, d)
    out = torch.zeros_like(q)
    spans = [(1 if n else 0, n - 1 if n else 0) for n in _lengths(case)] if case["kind"] == "decode" else _portions(case)
    t0 = 0
    for r, (n, cached) in enumerate(spans):
        total = n + cached
        if total:
            p = s["table"][r, :-(-total // page)].long()
            hidden = torch.arange(total, device=DEV)[None] > torch.arange(cached, total, device=DEV)[:, None]
            for kvh in range(nkv):
                k, v = (_places(s["kv"][p, kvh, i], page, d, bool(i)).reshape(-1, d)[:total] for i in range(2))
                for head in range(kvh * group, (kvh + 1) * group):
                    e = torch.where(hidden, -math.inf, (q[t0:t0 + n, head] @ k.T) / math.sqrt(d))
                    e = torch.exp(e - e.max(-1, keepdim=True)[0])
                    out[t0:t0 + n, head] = (e / e.sum(-1, keepdim=True)) @ v
        t0 += n if case["kind"] == "portions" else 1
    return out.view(-1, nq * d)
