"""What the comparison of portions over a 4-bit cache with 64 bits notices: mistakes planted in a statement in plain operations, on the CPU."""

import math

import pytest
import torch

import four_bits as fb
import four_bits_portions as fp
from four_bits import BF16, F32

F16 = torch.float16


def stated(q, kv, table, n, cached, nq, nkv, d, page, scale, keys=F16, weights=F16, values=F16, short=0):
    """The kernels' roundings: keys, weights (of up to 2^14) and values to the types given, all else in 64 bits; ``short``: keys that the causal mask hides too many."""
    total = n + cached
    out, x = torch.zeros(n, nq, d, dtype=torch.float64), q.double().view(n, nq, d)
    pages = table[0].long()[:-(-total // page)]
    hidden = torch.arange(total)[None] + short > torch.arange(cached, total)[:, None]
    for h in range(nq):
        k, v = (lo + s * c for c, s, lo in ([t.reshape(-1, d)[:total] for t in fb.read_rows(kv[pages, h // (nq // nkv), i], page, d, bool(i))] for i in range(2)))
        e = (x[:, h] @ k.to(keys).double().T * scale).masked_fill(hidden, -math.inf)
        p = torch.exp(e - e.amax(-1, keepdim=True)) * 2.0 ** 14
        out[:, h] = p.to(weights).double() @ v.to(values).double() / p.sum(-1, keepdim=True)
    return out.view(n, nq * d).to(BF16)


@pytest.mark.parametrize("nq,nkv,d,page", [(8, 2, 128, 64), (4, 4, 64, 16), (4, 1, 256, 64), (3, 1, 192, 8)])
@pytest.mark.parametrize("n,cached", [(300, 700), (130, 0), (64, 40)])
def test_mistakes_are_noticed(nq, nkv, d, page, n, cached):
    g = torch.Generator().manual_seed(n + d)
    table, pages = fb.tables([n + cached], page, g)
    kv = fb.random_cache(pages, nkv, page, d, g)
    q = torch.randn(n, nq * d, generator=g).to(BF16)
    out, bound = fp.want(q, kv, table, [(n, cached)], nq, nkv, d, page, d ** -0.5)
    run = lambda scale=d ** -0.5, **kw: fp.faults(stated(q, kv, table, n, cached, nq, nkv, d, page, scale, **kw), out, bound)
    assert run() == [] and run(keys=F32, weights=F32, values=F32) == []
    assert len(fp.faults(torch.zeros_like(out), out, bound)) == 2
    if cached:
        assert run(short=1)                               # (a first token that sees nothing has no softmax)
    for scale in (0.95, 1.05):
        assert run(scale * d ** -0.5)
    for what in ("keys", "values", *(("weights",) if cached else ())):      # (most of a prompt's norm is its first tokens', whose one or two weights are nearly 1 together)
        assert run(**{what: BF16}), what
