"""Plain statements of numbers held in four bits, in 64 bits and from the definitions: what codes stand for, what a cache holds, products and attention over them.
They run where their tensors are and share no code with the kernels' package."""

import math

import torch

F32, BF16 = torch.float32, torch.bfloat16
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}            # a rounding is off by at most this, relative to the value


def make_matrix(n, k, group, zeros, g, device="cpu"):
    """(codes [n, k], scales [n, k / group], zero points or None) of a random matrix."""
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = (torch.rand(n, k // group, generator=g) * 0.05 + 1e-3).to(BF16)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    return codes.to(device), scales.to(device), None if z is None else z.to(device)


def matrix_values(codes, scales, zeros):
    group = codes.shape[1] // scales.shape[1]
    wide = lambda t: t.double().repeat_interleave(group, 1)
    return wide(scales) * (codes.double() - (8.0 if zeros is None else wide(zeros)))


# ---- the cache: uint8 [pages, nkv, 2, page (d / 2 + d / 16)] ----

def code_place(d, value):
    """(byte, shift) of feature f's code in a place's row."""
    f = torch.arange(d)
    j, word, i = f // 64, f % 64 // 8, f % 8
    word = word * (d // 64) + j if value else (word % 4) * 2 * (d // 64) + 2 * j + word // 4
    return 4 * word + i // 2, (4 * (i % 2)).int()


def read_rows(rows, page, d, value):
    """(codes, steps, lowest) of cache rows [..., page (d / 2 + d / 16)], the codes [..., page, d] and the others [..., page, d] in 64 bits."""
    at, shift = (t.to(rows.device) for t in code_place(d, value))
    codes = (rows[..., :page * d // 2].reshape(*rows.shape[:-1], page, d // 2)[..., at].int() >> shift) & 15
    held = rows[..., page * d // 2:].contiguous().view(BF16).double().reshape(*rows.shape[:-1], page, d // 64, 2).repeat_interleave(64, -2)
    return codes.double(), held[..., 0], held[..., 1]


def write_row(rows, slot, page, d, value, codes, held):
    """Puts codes [d] and (step, lowest) pairs [d / 64, 2] at ``slot`` of one page's row of one head and kind, uint8 [page (d / 2 + d / 16)]."""
    at, shift = (t.to(rows.device) for t in code_place(d, value))
    out = torch.zeros(d // 2, dtype=torch.int32, device=rows.device)
    out.index_add_(0, at, codes.int() << shift)
    rows[slot * d // 2:(slot + 1) * d // 2] = out.to(torch.uint8)
    start = page * d // 2 + slot * d // 16
    rows[start:start + d // 16] = held.contiguous().view(torch.uint8).flatten()


def hold(x):
    """Heads [..., d] float32 as (codes, (step, lowest) pairs [..., d / 64, 2]), one IEEE operation after the other."""
    x = x.float().unflatten(-1, (-1, 64))
    low, high = x.amin(-1), x.amax(-1)
    step, low = ((high - low) * torch.tensor(1.0 / 15.0, dtype=F32, device=x.device)).to(BF16), low.to(BF16)
    bad = ~(torch.isfinite(step) & torch.isfinite(low))
    step, low = step.masked_fill(bad, math.nan), low.masked_fill(bad, math.nan)
    code = torch.round((x - low.float()[..., None]) / step.float()[..., None]).clamp(0, 15)
    return torch.where((step > 0)[..., None], code, 0.0).to(torch.uint8).flatten(-2), torch.stack([step, low], -1)


def turn(x, gain, eps, cos, sin, rot):
    """Norm and rotation of heads [tokens, heads, d] float32 as the cache's writer does them; cos, sin [tokens, rot / 2]."""
    if gain is not None:
        x = x * (1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + eps)).float() * gain.float()
    if not rot:
        return x
    a, b, cos, sin = x[..., :rot // 2], x[..., rot // 2:rot], cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def attention(q, kv, table, spans, nq, nkv, d, page, scale):
    """Causal attention in 64 bits of ``spans`` [(new, cached)], rows of q in their order: (outputs, bounds of what one rounding of the weights times steps, around the middle code 8, and of a value, moves them by)
    [tokens, nq * d].  A request without places has a row of zeros where it brings one token (``new`` 0)."""
    group, q = nq // nkv, q.double().view(-1, nq, d)
    out, by_codes, by_values = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    t0 = 0
    for r, (n, cached) in enumerate(spans):
        total = n + cached
        rows = max(n, 1)
        if n:
            pages = table[r].long()[:-(-total // page)]
            hidden = torch.arange(total, device=q.device)[None] > torch.arange(cached, total, device=q.device)[:, None]
            for kvh in range(nkv):
                (kc, ks, kl), (vc, vs, vl) = ([t.reshape(-1, d)[:total] for t in read_rows(kv[pages, kvh, i], page, d, bool(i))] for i in range(2))
                k, v = kl + ks * kc, vl + vs * vc
                for h in range(kvh * group, (kvh + 1) * group):
                    e = (q[t0:t0 + n, h] @ k.T * scale).masked_fill(hidden, -math.inf)
                    p = torch.softmax(e, -1)
                    out[t0:t0 + n, h] = p @ v
                    by_codes[t0:t0 + n, h] = p @ (vs * (vc - 8).abs())
                    by_values[t0:t0 + n, h] = p @ v.abs()
        t0 += rows
    return tuple(t.view(-1, nq * d) for t in (out, by_codes, by_values))


def random_cache(pages, nkv, page, d, g, lean=0.0):
    """A cache whose every page holds random numbers' codes, on the CPU; ``lean`` gives keys a common part of a size of their own."""
    x = torch.randn(pages, nkv, 2, page, d, generator=g)
    x[:, :, 0] += lean * torch.randn(pages, nkv, page, 1, generator=g)
    codes, held = hold(x)
    rows = []
    for value in (False, True):
        at, shift = code_place(d, value)
        c = codes[:, :, int(value)].int() << shift
        out = torch.zeros(pages, nkv, page, d // 2, dtype=torch.int32).index_add_(-1, at, c).to(torch.uint8)
        rows.append(torch.cat([out.flatten(-2), held[:, :, int(value)].contiguous().view(torch.uint8).flatten(-3)], -1))
    return torch.stack(rows, 2).contiguous()


def tables(lengths, page, g):
    """(block table int32 over shuffled pages, pages of the pool); page 0 belongs to nobody."""
    counts = [-(-n // page) for n in lengths]
    order = (torch.randperm(sum(counts) + 2, generator=g) + 1).int()
    table = torch.zeros(len(lengths), max(1, max(counts, default=1)), dtype=torch.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = order[at:at + c]
        at += c
    return table, sum(counts) + 3
