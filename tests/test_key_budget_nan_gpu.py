"""Tokens whose queries are no numbers: what they give to the keys they see is NaN, and they give nothing to those behind them."""

import math

import pytest
import torch

from test_key_budget_gpu import BF16, DEV, F32, close, pool, portion_want, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d,page", [(F32, 64, 16), (F32, 40, 64), (BF16, 48, 16), (BF16, 64, 64), (BF16, 128, 16)])
@pytest.mark.parametrize("nq,nkv", [(4, 2), (14, 2), (3, 3)])
@pytest.mark.parametrize("cached,n,token", [(0, 300, 3), (0, 300, 70), (100, 200, 0), (37, 90, 40), (0, 65, 64)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_token_without_a_number_gives_nothing_to_the_keys_behind_it(dtype, d, page, nq, nkv, cached, n, token, value):
    from lily_b200.csrc import ops
    kv, w, table = pool([cached + n], nkv, page, d, dtype, 3, lean=0.3)
    q = torch.randn(n, nq * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).to(dtype)
    want = rows_of(portion_want(q, kv, w, table, [cached], [n], nq, nkv, d, page, d ** -0.5, None), table, 0, cached + n, page)
    q[token] = value                                              # (infinite in all features: scores of both signs, whose softmax is none)
    cu, pre = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.tensor([cached], dtype=torch.int32, device=DEV)
    ops.attention_key_weights(q, kv, w, table, cu, pre, [cached], [n], nq, nkv, d, page, d ** -0.5)
    got, seen = rows_of(w, table, 0, cached + n, page), cached + token + 1
    if math.isnan(value):
        assert bool(torch.isnan(got[:, :seen]).all())
    close(got[:, seen:], want[:, seen:], F32)
