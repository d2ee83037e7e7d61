"""What lies outside the tables of a budgeted cache is neither read nor written."""

import pytest
import torch

from test_key_budget_gpu import BF16, DEV, F32, pool, same

pytestmark = pytest.mark.gpu


def ops():
    from lily_b200.csrc import ops as o
    return o


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [128, 80])
@pytest.mark.parametrize("planes", [0, 2])
def test_tokens_of_no_request_are_not_written(dtype, d, planes):
    """Requests ahead of the block table and behind it (padding, a request that has gone): the queries come out, the cache stays."""
    nq, nkv, page, n = 4, 2, 16, 7
    kv, _, table = pool([40, 20], nkv, page, d, dtype, 6)
    g = torch.Generator(device=DEV).manual_seed(3)
    shape = (n, (nq + 2 * nkv) * d)
    qkv = torch.randn(planes, *shape, device=DEV, generator=g) if planes else torch.randn(shape, device=DEV, generator=g).to(dtype)
    angle = torch.rand(50, d // 2, device=DEV, generator=g)
    positions = torch.arange(n, dtype=torch.int32, device=DEV).expand(2, n).contiguous()
    places = torch.arange(n, dtype=torch.int32, device=DEV)
    write = lambda req, cache: ops().axes_rope_write(qkv, None, None, 1e-6, angle.cos(), angle.sin(), positions, ops().pair_axes((d // 4, d // 2 - d // 4), DEV), places,
                                                     torch.tensor(req, dtype=torch.int32, device=DEV), table, cache, nq, nkv, d, d, page)
    whole, some = kv.clone(), kv.clone()
    want = write([0, 1, 0, 1, 0, 1, 0], whole)
    got = write([0, -1, 2, 1, 1 << 30, -(1 << 31), 0], some)
    assert torch.equal(got, want)
    for place in (1, 2, 4, 5):                                    # those whose request is none
        for r in range(2):
            at = table[r, place // page].long()
            whole[at, :, :, place % page] = kv[at, :, :, place % page]
    assert same(some, whole) and not same(some, kv)
