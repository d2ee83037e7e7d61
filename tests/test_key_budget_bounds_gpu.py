"""What lies outside the tables of a budgeted cache is neither read nor written."""

import pytest
import torch

from test_key_budget_gpu import BF16, DEV, F32, pool, rows_of, same

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


@pytest.mark.parametrize("dtype,d", [(F32, 128), (BF16, 128), (BF16, 80)])
def test_pages_of_any_size_hold_the_same_places(dtype, d):
    """Places are found by a shift where a page is a power of two, by a quotient elsewhere."""
    nq, nkv, new = 4, 2, [40, 27]
    n = sum(new)
    g = torch.Generator(device=DEV).manual_seed(3)
    qkv = torch.randn(n, (nq + 2 * nkv) * d, device=DEV, generator=g).to(dtype)
    angle = torch.rand(50, d // 2, device=DEV, generator=g)
    positions = torch.randint(0, 50, (1, n), dtype=torch.int32, device=DEV, generator=g)
    places = torch.cat([torch.arange(m) for m in new]).int().to(DEV)
    req = torch.repeat_interleave(torch.arange(2), torch.tensor(new)).int().to(DEV)
    held = []
    for page in (16, 12, 7, 1):
        kv, _, table = pool(new, nkv, page, d, dtype, 6)
        q = ops().axes_rope_write(qkv, None, None, 1e-6, angle.cos(), angle.sin(), positions, ops().pair_axes((d // 2,), DEV), places, req, table, kv, nq, nkv, d, d, page)
        held.append([q] + [rows_of(kv[:, i], table, r, m, page) for r, m in enumerate(new) for i in range(2)])
    for other in held[1:]:
        assert all(torch.equal(a, b) for a, b in zip(held[0], other))
    want = qkv.view(n, -1, d)[:, nq + nkv:]                       # values are what came
    assert torch.equal(held[0][2], want[:new[0]].transpose(0, 1).double()) and torch.equal(held[0][4], want[new[0]:].transpose(0, 1).double())
