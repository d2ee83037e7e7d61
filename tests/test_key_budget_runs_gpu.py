"""Column sums of prompt portions on the CUDA cores, whose scores come in runs of tokens where a portion has many: against 64 bits, with
scratch that holds NaN, so that nothing may be read that was not written."""

import math

import pytest
import torch

from test_key_budget_gpu import BF16, DEV, F32, close, pool, portion_want, same

pytestmark = pytest.mark.gpu


def ops():
    from lily_b200.csrc import ops as o
    return o


def given(q, kv, w, table, cached, new, nq, nkv, d, page, observe):
    """What the call makes of a copy of ``w``, its scratch filled with NaN."""
    w, o = w.clone(), ops()
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    pre = torch.tensor(cached, dtype=torch.int32, device=DEV)
    scratch = torch.full((o.key_weights_scratch_floats(cached, new, nq, nkv, d, page, d ** -0.5, q.dtype, observe),), math.nan, device=DEV)
    o.attention_key_weights(q, kv, w, table, cu, pre, cached, new, nq, nkv, d, page, d ** -0.5, observe=observe, scratch=scratch)
    return w


def portions(cached, new, nq, nkv, d, page, dtype, seed):
    kv, w, table = pool([p + n for p, n in zip(cached, new)], nkv, page, d, dtype, seed, lean=0.3)
    for r, (p, n) in enumerate(zip(cached, new)):                 # what the portion's own places hold is nobody's
        for j in range(p, p + n):
            w[table[r, j // page].long(), :, j % page] = math.nan
    q = torch.randn(sum(new), nq * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(dtype)
    return q, kv, w, table


@pytest.mark.parametrize("dtype,d,page", [(F32, 64, 16), (BF16, 48, 64)])
@pytest.mark.parametrize("nq,nkv", [(3, 3), (6, 2), (8, 2), (7, 1)])
@pytest.mark.parametrize("cached,new,observe", [([0], [500], None), ([0, 129, 40], [333, 70, 200], None), ([300, 7], [411, 260], 190), ([64], [333], None)])
@pytest.mark.parametrize("run", [64, 71, 100, 250])
def test_portions_in_several_runs(monkeypatch, dtype, d, page, nq, nkv, cached, new, observe, run):
    """Two to eight runs of ``run`` tokens, of which a tile of 64 rows, heads below one another, is seldom full at the end."""
    q, kv, w, table = portions(cached, new, nq, nkv, d, page, dtype, 4)
    want = portion_want(q, kv, w, table, cached, new, nq, nkv, d, page, d ** -0.5, observe)
    whole = given(q, kv, w, table, cached, new, nq, nkv, d, page, observe)
    monkeypatch.setattr(ops(), "KEY_WEIGHTS_SCORES", run * nq * sum(p + n + 64 for p, n in zip(cached, new)))
    got = given(q, kv, w, table, cached, new, nq, nkv, d, page, observe)
    close(whole, want, F32)
    close(got, want, F32)
    assert same(got, given(q, kv, w, table, cached, new, nq, nkv, d, page, observe))


@pytest.mark.parametrize("cached,new,nq,nkv", [(0, 5042, 32, 8), (700, 4000, 16, 4)])
def test_a_portion_that_is_too_long_for_one_run(cached, new, nq, nkv):
    """The runs that the sizes ask for by themselves: 1,642 and 3,521 tokens."""
    d, page = 64, 64
    q, kv, w, table = portions([cached], [new], nq, nkv, d, page, F32, 5)
    want = portion_want(q, kv, w, table, [cached], [new], nq, nkv, d, page, d ** -0.5, None)
    close(given(q, kv, w, table, [cached], [new], nq, nkv, d, page, None), want, F32)
