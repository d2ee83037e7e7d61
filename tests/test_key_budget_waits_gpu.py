"""Waits of the tcgen05 column sums that run out: what is void is NaN, the host hears of it once, and the next call is as before."""

import math

import pytest
import torch

from test_key_budget_gpu import BF16, DEV, close, F32, pool, portion_want, rows_of, same

pytestmark = pytest.mark.gpu
PLENTY = 1 << 24


@pytest.mark.parametrize("polls", [(0, PLENTY), (PLENTY, 0), (0, 0)])
@pytest.mark.parametrize("nq,nkv,d,page", [(8, 2, 128, 64), (14, 2, 64, 16), (3, 3, 64, 8)])
@pytest.mark.parametrize("cached,new,observe", [([0], [1], None), ([0, 300, 5], [700, 0, 90], None), ([3000, 40], [130, 77], 16), ([0], [2500], None)])
def test_a_wait_that_runs_out_makes_the_weights_void_and_nothing_else(monkeypatch, polls, nq, nkv, d, page, cached, new, observe):
    """No polls at all in the row kernel, the column kernel, both: every block gives up.  (One block a tile, and tiles that several share.)"""
    from lily_b200.csrc import ops as o
    lengths = [p + n for p, n in zip(cached, new)]
    kv, w, table = pool(lengths, nkv, page, d, BF16, 3, lean=0.3)
    q = torch.randn(sum(new), nq * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(BF16)
    want = portion_want(q, kv, w, table, cached, new, nq, nkv, d, page, d ** -0.5, observe)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    pre = torch.tensor(cached, dtype=torch.int32, device=DEV)

    def run():
        mine = w.clone()
        o.attention_key_weights(q, kv, mine, table, cu, pre, cached, new, nq, nkv, d, page, d ** -0.5, observe=observe)
        torch.cuda.synchronize()
        return mine
    first = run()
    close(first, want, F32)
    assert o.key_weights_lost() == 0
    monkeypatch.setattr(o, "KEY_WEIGHTS_POLLS", polls)
    void = run()
    assert o.key_weights_lost() >> 24 in range(1, 10) and o.key_weights_lost() == 0 and o.key_weights_status() == 0
    expected = w.clone()
    for r, (p, n) in enumerate(zip(cached, new)):
        if n:
            assert bool(torch.isnan(rows_of(void, table, r, p + n, page)).all())
            for j in range(p + n):
                expected[table[r, j // page].long(), :, j % page] = math.nan
    assert same(void, expected)                                   # requests without tokens, and all that lies outside
    monkeypatch.undo()
    assert same(run(), first) and o.key_weights_status() == 0


def test_a_void_call_on_one_stream_leaves_another_call_alone(monkeypatch):
    """Nothing of a call whose waits ran out is kept on the device: a call that nobody asked about in between is right."""
    from lily_b200.csrc import ops as o
    nq, nkv, d, page, n = 8, 2, 128, 64, 600
    kv, w, table = pool([n], nkv, page, d, BF16, 3)
    q = torch.randn(n, nq * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(BF16)
    cu, pre = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    run = lambda mine: o.attention_key_weights(q, kv, mine, table, cu, pre, [0], [n], nq, nkv, d, page, d ** -0.5)
    want, void, after = w.clone(), w.clone(), w.clone()
    run(want)
    monkeypatch.setattr(o, "KEY_WEIGHTS_POLLS", (0, PLENTY))
    run(void)
    monkeypatch.undo()
    run(after)
    assert same(after, want) and not same(void, want) and o.key_weights_status() != 0
