"""What the operators of a budgeted key/value cache are measured on.

A long request's cache is held to a budget of places: attention says what weight each cached key was given, and the keys that were
given the least are let go of.  A token's place in the cache is then no longer its position, so the kernel that writes keys takes both,
and the position may have several axes (time, height, width), as in prompts with images.  Four kinds of case:

* ``write``    per-head norm, rotation by positions with several axes, queries out, keys and values to their places in the pages.
* ``decode``   attention of one new token a request over its pages, which also adds up the weight every cached place was given.
* ``weights``  what a prompt's portion (``n@p``: n tokens behind p cached ones; or its last ``observe`` tokens) gives to every place.
* ``evict``    in all layers of a cache: choose the places each kv head keeps, and move their keys, values and weights to the front of
               the pages of a fork of the request (the whole prompt stays cached for others).

Sizes are those of ``perf/cases.py``: "small" (16 query heads over 4 kv heads of 128) and "mid" (32 over 8), pages of 64 or 16.
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
TABLE = 32768                    # positions in the rotation tables


def listed():
    return [
        # a decode step of eight users: the projection's float32 partial sums become queries and one cached row each
        {"name": "write-8", "kind": "write", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "rot": 128, "page": 64, "tokens": "1,1,1,1,1,1,1,1", "planes": 4, "norm": True, "mixed": False},
        # a prompt of text around an image, three axes in runs of pairs
        {"name": "write-2048", "kind": "write", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "rot": 128, "page": 64, "tokens": "2048", "planes": 0, "norm": True, "mixed": False},
        # the 32-bit path: ragged prompts, half of a head rotated, axes in turn, no norm
        {"name": "write-f32", "kind": "write", "dtype": "f32", "nq": 16, "nkv": 4, "d": 128, "rot": 64, "page": 16, "tokens": "703,1,399", "planes": 0, "norm": False, "mixed": True},
        # one user of a small model, short context: the smallest call
        {"name": "decode-1", "kind": "decode", "dtype": "bf16", "nq": 16, "nkv": 4, "d": 128, "page": 64, "rows": 1, "low": 900, "high": 900},
        # eight users at 4,096 places
        {"name": "decode-8", "kind": "decode", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "page": 64, "rows": 8, "low": 4096, "high": 4096},
        # a busy server: 64 users with caches of very different lengths
        {"name": "decode-64", "kind": "decode", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "page": 64, "rows": 64, "low": 250, "high": 1750},
        # checking a checkpoint in 32-bit
        {"name": "decode-f32", "kind": "decode", "dtype": "f32", "nq": 16, "nkv": 4, "d": 128, "page": 16, "rows": 3, "low": 150, "high": 2900},
        # one prompt whose every token is heard
        {"name": "weights-2048", "kind": "weights", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "page": 64, "portions": "2048", "observe": 0},
        # the end of a long prompt, whose last 64 tokens are heard
        {"name": "weights-16k", "kind": "weights", "dtype": "bf16", "nq": 32, "nkv": 8, "d": 128, "page": 64, "portions": "1024@15360", "observe": 64},
        # ragged portions in 32-bit, one of them a single token
        {"name": "weights-f32", "kind": "weights", "dtype": "f32", "nq": 16, "nkv": 4, "d": 128, "page": 16, "portions": "333,70@300,1@511", "observe": 0},
        # one request brought from 4,096 places to 1,024 in eight layers
        {"name": "evict-1", "kind": "evict", "dtype": "bf16", "layers": 8, "nkv": 8, "d": 128, "page": 64, "rows": 1, "low": 4096, "high": 4096, "keep": 1024, "first": 4, "recent": 128},
        # many requests at once, some of them already within the budget
        {"name": "evict-24", "kind": "evict", "dtype": "bf16", "layers": 4, "nkv": 4, "d": 128, "page": 64, "rows": 24, "low": 400, "high": 3500, "keep": 512, "first": 4, "recent": 64},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["write", "decode", "weights", "evict"])
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    nq, nkv, d = rng.choice([(16, 4, 128), (32, 8, 128), (16, 16, 64), (12, 4, 64), (14, 2, 64), (16, 2, 128)])
    page = rng.choice([16, 64, 64])
    c = {"kind": kind, "dtype": dtype, "nq": nq, "nkv": nkv, "d": d, "page": page}
    if kind == "write":
        rows = rng.random() < 0.4
        c["tokens"] = ",".join(["1"] * _log(rng, 1, 64)) if rows else ",".join(str(_log(rng, 2, 680)) for _ in range(rng.randint(1, 3)))
        c.update(rot=d if rng.random() < 0.7 else d // 2, planes=rng.choice([0, 2, 5]) if rows else 0, norm=rng.random() < 0.6, mixed=rng.random() < 0.5)
    elif kind == "decode":
        c["rows"] = _log(rng, 1, 48)
        c["high"] = _log(rng, 1, min(32768, 60000 // c["rows"]) // (4 if dtype == "f32" else 1))
        c["low"] = _log(rng, max(1, c["high"] // 8), c["high"])
    elif kind == "weights":
        several = rng.randint(1, 3)
        top = 500 if dtype == "f32" else 1100
        c["portions"] = ",".join(f"{_log(rng, 1, top)}@{rng.choice([0, _log(rng, 1, 2 * top)])}" for _ in range(several))
        c["observe"] = rng.choice([0, 0, _log(rng, 1, 100)])
    else:
        c.pop("nq")
        c.update(layers=rng.randint(1, 6), rows=_log(rng, 1, 12), high=_log(rng, 8, 6000))
        c["high"] = max(8, min(c["high"], 24000 // c["rows"]))
        c["low"] = _log(rng, max(4, c["high"] // 6), c["high"])
        c["keep"] = _log(rng, 4, c["high"])
        c["first"] = rng.randint(0, min(4, c["keep"] // 2))
        c["recent"] = rng.randint(0, c["keep"] // 2)
    return c


def _lengths(case):
    """``rows`` lengths spread between ``low`` and ``high`` (both among them)."""
    n, low, high = case["rows"], case["low"], case["high"]
    if n == 1:
        return [high]
    return [round(low * (high / low) ** ((i * 5 % n if n % 5 else i) / (n - 1))) for i in range(n)]


def _portions(case):
    """(new, cached) of every portion."""
    return [tuple(int(x) for x in (p.split("@") + ["0"])[:2]) for p in case["portions"].split(",")]


def work(case):
    item = 2 if case["dtype"] == "bf16" else 4
    d, nkv = case["d"], case["nkv"]
    if case["kind"] == "write":
        n = sum(int(x) for x in case["tokens"].split(","))
        row = (case["nq"] + 2 * nkv) * d
        read = row * (4 * case["planes"] if case["planes"] else item)
        return {"bytes": n * (read + row * item + 4 * case["rot"]), "flops": n * row * 6}
    if case["kind"] == "decode":
        places = sum(_lengths(case))
        return {"bytes": places * nkv * (2 * d * item + 8) + case["rows"] * case["nq"] * d * 2 * item, "flops": 4 * places * case["nq"] * d}
    if case["kind"] == "weights":
        moved = pairs = 0
        for n, p in _portions(case):
            heard = min(n, case["observe"] or n)
            pairs += sum(p + t + 1 for t in range(n - heard, n))
            moved += heard * case["nq"] * d * item + (p + n) * nkv * (d * item + 4) + p * nkv * 4
        return {"bytes": moved, "flops": 2 * pairs * case["nq"] * d}
    lengths = _lengths(case)
    kept = sum(min(n, case["keep"]) for n in lengths)
    return {"bytes": case["layers"] * nkv * (4 * sum(lengths) + kept * (4 + 8 + 4 * d * item)), "flops": case["layers"] * nkv * sum(lengths)}


# ------------------------------------------------------------------------------ what a program has in hand

def _pages(lengths, page, g):
    """Block tables over shuffled pages, and the pages of the pool (page 0 belongs to nobody)."""
    counts = [-(-n // page) for n in lengths]
    total = sum(counts) + 3
    order = torch.randperm(total, generator=g)[:sum(counts)] + 1
    table = torch.nn.utils.rnn.pad_sequence(order.split(counts), batch_first=True)
    return table.int().contiguous().to(DEV), total


def _image_prompt(n, start):
    """Positions [3, n] of a quarter of text, an image (one time, rows and columns), then text."""
    text, image = n // 4, n // 2
    i, side = torch.arange(image), max(1, math.isqrt(image))
    grid = start + text + torch.stack([torch.zeros_like(i), i // side, i % side])
    last = int(grid.max()) + 1 if image else start + text
    return torch.cat([(start + torch.arange(text)).expand(3, -1), grid, (last + torch.arange(n - text - image)).expand(3, -1)], 1)


def prepare(case, seed):
    h = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    nkv, d, page = case["nkv"], case["d"], case["page"]
    s = {"case": case, "dtype": dtype}
    if case["kind"] == "write":
        tokens = [int(x) for x in case["tokens"].split(",")]
        n, nq, rot = sum(tokens), case["nq"], case["rot"]
        cached = [(37 * i + 5) % (3 * page) for i in range(len(tokens))]
        s["table"], pages = _pages([c + t for c, t in zip(cached, tokens)], page, h)
        s["kv"] = torch.randn(pages + 1, 2, nkv, page, d, device=DEV, generator=g).to(dtype)
        row = (nq + 2 * nkv) * d
        if case["planes"]:
            s["qkv"] = torch.randn(case["planes"], n, row, device=DEV, generator=g)
        else:
            s["qkv"] = torch.randn(n, row, device=DEV, generator=g).to(dtype)
        s["gains"] = [(1 + 0.2 * torch.randn(d, device=DEV, generator=g)).to(dtype) for _ in range(2)] if case["norm"] else [None, None]
        inv = 1.0 / 10000.0 ** (torch.arange(0, rot, 2, dtype=torch.float32) / rot)
        angle = torch.outer(torch.arange(TABLE, dtype=torch.float32), inv)
        s["cos"], s["sin"] = angle.cos().to(DEV), angle.sin().to(DEV)
        half = rot // 2
        runs = [half // 4, half // 4 + half // 8]
        axis = torch.arange(half) % 3 if case["mixed"] else torch.tensor([0] * runs[0] + [1] * runs[1] + [2] * (half - sum(runs)))
        s["axis"] = axis.int().to(DEV)
        start = torch.randint(0, TABLE - 4100, (len(tokens),), generator=h).tolist()
        s["positions"] = torch.cat([_image_prompt(t, at) for t, at in zip(tokens, start)], 1).int().to(DEV)
        s["places"] = torch.cat([c + torch.arange(t) for c, t in zip(cached, tokens)]).int().to(DEV)
        s["req"] = torch.repeat_interleave(torch.arange(len(tokens)), torch.tensor(tokens)).int().to(DEV)
        return s
    if case["kind"] == "evict":
        lengths = _lengths(case)
        keep = case["keep"]
        room = [min(n, keep) for n in lengths]
        both, pages = _pages(lengths + room, page, h)
        s["table"], s["to"] = both[:len(lengths)].contiguous(), both[len(lengths):, :max(1, -(-max(room) // page))].contiguous()
        s["kv"] = torch.randn(case["layers"], pages + 1, 2, nkv, page, d, device=DEV, generator=g, dtype=dtype)
        w = torch.randn(case["layers"], pages + 1, nkv, page, device=DEV, generator=g).mul_(2).exp_()
        s["weights"] = torch.where(w < 0.1, torch.floor(w * 40) / 40, w)           # rarely seen places tie, many of them at zero
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        s["longest"] = max(lengths)
        return s
    nq = case["nq"]
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
    lean = torch.randn(nkv, d, device=DEV, generator=g) / math.sqrt(d)
    kv = torch.randn(pages + 1, 2, nkv, page, d, device=DEV, generator=g)
    heavy = torch.randn(pages + 1, nkv, page, device=DEV, generator=g).exp() * 1.5        # how far a key leans the queries' way
    kv[:, 0] += heavy[..., None] * lean[:, None]
    s["kv"] = kv.to(dtype)
    q = torch.randn(sum(new), nkv, nq // nkv, d, device=DEV, generator=g) + 3 * lean[:, None]
    s["q"] = q.reshape(sum(new), nq * d).to(dtype)
    s["weights"] = torch.rand(pages + 1, nkv, page, device=DEV, generator=g) * 3
    return s


# ------------------------------------------------------------------------------ one pass

def run(s):
    return (_own if own else _plain)[s["case"]["kind"]](s)


def _own_write(s):
    from lily_b200.csrc import ops
    c = s["case"]
    q = ops.axes_rope_write(s["qkv"], *s["gains"], EPS, s["cos"], s["sin"], s["positions"], s["axis"], s["places"], s["req"], s["table"],
                            s["kv"], c["nq"], c["nkv"], c["d"], c["rot"], c["page"])
    return {"q": q, "kv": s["kv"]}


def _own_decode(s):
    from lily_b200.csrc import ops
    c = s["case"]
    out = ops.attention_decode_weighed(s["q"], s["kv"], s["weights"], s["table"], s["seq_lens"], s["longest"], c["nq"], c["nkv"], c["d"],
                                       c["page"], c["d"] ** -0.5)
    return {"out": out, "weights": s["weights"]}


def _own_weights(s):
    from lily_b200.csrc import ops
    c = s["case"]
    ops.attention_key_weights(s["q"], s["kv"], s["weights"], s["table"], s["cu"], s["prefix"], s["cached"], s["new"], c["nq"], c["nkv"],
                              c["d"], c["page"], c["d"] ** -0.5, observe=c["observe"] or None)
    return {"weights": s["weights"]}


def _own_evict(s):
    from lily_b200.csrc import ops
    c = s["case"]
    kept = ops.select_keys(s["weights"], s["table"], s["lengths"], s["longest"], c["keep"], c["first"], c["recent"])
    ops.move_keys(s["kv"], s["weights"], s["table"], kept, to_table=s["to"])
    return {"kept": kept, "kv": s["kv"], "weights": s["weights"]}


def _turn(x, gain, cos, sin, rot):
    """Norm of the last axis where there is a gain, then rotation of its first ``rot`` features by halves."""
    if gain is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gain.float()
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def _plain_write(s):
    c = s["case"]
    nq, nkv, d, page, rot = c["nq"], c["nkv"], c["d"], c["page"], c["rot"]
    x = s["qkv"].sum(0) if c["planes"] else s["qkv"].float()
    x = x.view(x.shape[0], nq + 2 * nkv, d)
    pair = torch.arange(rot // 2, device=x.device)
    at = s["positions"].long()[s["axis"].long()].t()                                # [tokens, pairs]
    cos, sin = s["cos"][at, pair][:, None], s["sin"][at, pair][:, None]
    q = _turn(x[:, :nq], s["gains"][0], cos, sin, rot).reshape(-1, nq * d).to(s["dtype"])
    places = s["places"].long()
    pages = s["table"].long()[s["req"].long(), places // page]
    s["kv"][pages, 0, :, places % page] = _turn(x[:, nq:nq + nkv], s["gains"][1], cos, sin, rot).to(s["dtype"])
    s["kv"][pages, 1, :, places % page] = x[:, nq + nkv:].to(s["dtype"])
    return {"q": q, "kv": s["kv"]}


def _gather(s, longest):
    """(pages, offsets) of the places [0, longest) of every request."""
    j = torch.arange(longest, device=DEV)
    return s["table"].long()[:, j // s["case"]["page"]], j % s["case"]["page"]


def _plain_decode(s):
    c = s["case"]
    nq, nkv, d = c["nq"], c["nkv"], c["d"]
    pages, off = _gather(s, s["longest"])
    j = torch.arange(s["longest"], device=DEV)
    lengths = s["seq_lens"].long()[:, None]
    k, v = s["kv"][pages, 0, :, off].float(), s["kv"][pages, 1, :, off].float()       # [rows, places, kv heads, d]
    q = s["q"].float().view(-1, nkv, nq // nkv, d)
    scores = torch.einsum("rgnd,rlgd->rgnl", q, k) * d ** -0.5
    p = torch.softmax(scores.masked_fill((j >= lengths)[:, None, None], -math.inf), -1)
    out = torch.einsum("rgnl,rlgd->rgnd", p, v).reshape(-1, nq * d).to(s["dtype"])
    old = s["weights"][pages, :, off]                                                  # [rows, places, kv heads]
    add = p.sum(2).transpose(1, 2) + torch.where((j < lengths - 1)[..., None], old, 0.0)
    held = (j < lengths)[..., None]
    s["weights"][pages, :, off] = torch.where(held, add, old)
    return {"out": out, "weights": s["weights"]}


def _plain_weights(s):
    c = s["case"]
    nq, nkv, d = c["nq"], c["nkv"], c["d"]
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    longest = max(a + b for a, b in zip(s["new"], s["cached"]))
    heard = max(min(n, c["observe"] or n) for n in s["new"])
    pages, off = _gather(s, longest)
    j = torch.arange(longest, device=DEV)
    back = torch.arange(heard, device=DEV)                                             # row b is token new - 1 - b
    rows = (s["cu"][1:].long() - 1)[:, None] - back                                    # [requests, heard]
    is_row = back < new[:, None]
    q = s["q"].float()[rows.clamp(min=0)].view(-1, heard, nkv, nq // nkv, d)
    k = s["kv"][pages, 0, :, off].float()
    scores = torch.einsum("rtgnd,rlgd->rgntl", q, k) * d ** -0.5
    last = (s["prefix"].long() + new - 1)[:, None] - back                              # the place of each row's own token
    seen = j <= last[..., None]                                                        # [requests, heard, places]
    p = torch.softmax(scores.masked_fill(~seen[:, None, None], -math.inf).masked_fill(~is_row[:, None, None, :, None], 0.0), -1)
    add = (p * is_row[:, None, None, :, None]).sum((2, 3)).transpose(1, 2)
    old = s["weights"][pages, :, off]
    total = (s["prefix"].long() + new)[:, None]
    value = add + torch.where((j < s["prefix"].long()[:, None])[..., None], old, 0.0)
    s["weights"][pages, :, off] = torch.where((j < total)[..., None], value, old)
    return {"weights": s["weights"]}


def _plain_evict(s):
    c = s["case"]
    keep, page = c["keep"], c["page"]
    pages, off = _gather(s, s["longest"])
    j = torch.arange(s["longest"], device=DEV)
    n = s["lengths"].long()[:, None]
    w = s["weights"][:, pages, :, off].permute(2, 0, 3, 1)                             # [layers, requests, kv heads, places]
    sure = ((j < c["first"]) | (j >= n - c["recent"]))[None, :, None]
    w = torch.where(sure, math.inf, w).masked_fill((j >= n)[None, :, None], -math.inf)
    most = min(keep, s["longest"])
    at = torch.sort(w, dim=-1, descending=True, stable=True)[1][..., :most]
    at = torch.where(at < n[:, None], at, s["longest"])
    at = torch.sort(at, -1)[0]
    kept = torch.nn.functional.pad(torch.where(at < n[:, None], at, -1), (0, keep - most), value=-1).int()
    at = kept[..., :most].long()
    i = torch.arange(most, device=DEV)
    layer = torch.arange(c["layers"], device=DEV)[:, None, None, None]
    row = torch.arange(at.shape[1], device=DEV)[:, None, None]
    head = torch.arange(c["nkv"], device=DEV)[:, None]
    valid = at >= 0
    src = s["table"].long()[row, at.clamp(min=0) // page], at.clamp(min=0) % page
    dst = s["to"].long()[row, (i // page).expand(at.shape[1:])].expand(at.shape), (i % page).expand(at.shape)
    layer, head = layer.expand(at.shape), head.expand(at.shape)
    for_kv = valid[..., None, None]
    both = torch.arange(2, device=DEV)
    take = lambda p, o: s["kv"][layer[..., None], p[..., None], both, head[..., None], o[..., None]]
    moved = torch.where(for_kv, take(*src), take(*dst))
    s["kv"][layer[..., None], dst[0][..., None], both, head[..., None], dst[1][..., None]] = moved
    w = torch.where(valid, s["weights"][layer, src[0], head, src[1]], s["weights"][layer, dst[0], head, dst[1]])
    s["weights"][layer, dst[0], head, dst[1]] = w
    return {"kept": kept, "kv": s["kv"], "weights": s["weights"]}


_own = {"write": _own_write, "decode": _own_decode, "weights": _own_weights, "evict": _own_evict}
_plain = {"write": _plain_write, "decode": _plain_decode, "weights": _plain_weights, "evict": _plain_evict}


# ------------------------------------------------------------------------------ from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    d, nkv, page = case["d"], case["nkv"], case["page"]
    table = s["table"].tolist()
    if case["kind"] == "write":
        nq, rot = case["nq"], case["rot"]
        rows = s["qkv"].double()
        if case["planes"]:
            rows = rows.sum(0)
        heads = rows.view(len(rows), nq + 2 * nkv, d)
        cache = s["kv"].double()
        phase = torch.empty(len(rows), rot // 2, dtype=torch.complex128, device=DEV)
        for f, a in enumerate(s["axis"].tolist()):
            p = s["positions"][a].long()
            phase[:, f] = torch.complex(s["cos"][p, f].double(), s["sin"][p, f].double())
        done = []
        for part, gain in ((heads[:, :nq], s["gains"][0]), (heads[:, nq:nq + nkv], s["gains"][1])):
            x = part if gain is None else part / ((part * part).sum(-1, keepdim=True) / d + EPS).sqrt() * gain.double()
            z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * phase[:, None]
            done.append(torch.cat([z.real, z.imag, x[..., rot:]], -1))
        for t, (r, at) in enumerate(zip(s["req"].tolist(), s["places"].tolist())):
            p = table[r][at // page]
            cache[p, 0, :, at % page] = done[1][t]
            cache[p, 1, :, at % page] = heads[t, nq + nkv:]
        return {"q": done[0].reshape(len(rows), nq * d), "kv": cache}
    w = s["weights"].double()
    if case["kind"] == "evict":
        kept = torch.full((case["layers"], case["rows"], nkv, case["keep"]), -1, dtype=torch.int32)
        for r, n in enumerate(s["lengths"].tolist()):
            p = torch.tensor(table[r][:-(-n // page)], device=DEV)
            mine = w[:, p].transpose(1, 2).reshape(case["layers"], nkv, -1)[..., :n]
            if n > case["keep"]:
                middle = mine[..., case["first"]:n - case["recent"]]
                order = torch.argsort(-middle, dim=-1, stable=True)[..., :case["keep"] - case["first"] - case["recent"]] + case["first"]
                ends = torch.tensor([*range(case["first"]), *range(n - case["recent"], n)], device=DEV, dtype=torch.long)
                at = torch.cat([order, ends.expand(*order.shape[:2], len(ends))], -1).sort(-1)[0]
            else:
                at = torch.arange(n, device=DEV).expand(case["layers"], nkv, n)
            kept[:, r, :, :at.shape[-1]] = at.cpu().int()
            held = torch.gather(mine, -1, at)
            for i0 in range(0, at.shape[-1], page):
                part = held[..., i0:i0 + page]
                w[:, s["to"][r, i0 // page].long(), :, :part.shape[-1]] = part
        return {"kept": kept, "kv": None, "weights": w}
    nq = case["nq"]
    group = nq // nkv
    q = s["q"].double().view(-1, nq, d)
    out = torch.zeros_like(q)
    spans = [(1, n - 1) for n in _lengths(case)] if case["kind"] == "decode" else _portions(case)
    t0 = 0
    for r, (n, cached) in enumerate(spans):
        total, heard = n + cached, min(n, case.get("observe") or n)
        places = torch.arange(total, device=DEV)
        p = torch.tensor(table[r][:-(-total // page)], device=DEV)
        flat = lambda x: x.transpose(0, 1).reshape(nkv, -1, d)[:, :total].double()
        k, v = flat(s["kv"][p, 0]), flat(s["kv"][p, 1])
        own_place = torch.arange(total - heard, total, device=DEV)
        hidden = places[None] > own_place[:, None]
        for kvh in range(nkv):
            given = torch.zeros(total, dtype=torch.float64, device=DEV)
            for h in range(kvh * group, (kvh + 1) * group):
                e = (q[t0 + n - heard:t0 + n, h] @ k[kvh].T) / math.sqrt(d)
                e = torch.where(hidden, -math.inf, e)
                e = torch.exp(e - e.max(-1, keepdim=True)[0])
                e = e / e.sum(-1, keepdim=True)
                given += e.sum(0)
                if case["kind"] == "decode":
                    out[t0, h] = e[0] @ v[kvh]
            at = (p[places // page], kvh, places % page)
            w[at] = given + torch.where(places < cached, w[at], 0.0)
        t0 += n
    return {"out": out.view(-1, nq * d), "weights": w} if case["kind"] == "decode" else {"weights": w}
