"""Portions of prompts over a cache held in four bits against 64 bits, each output within what half precision moves it by and all together within their own rounding."""

import pytest
import torch

import four_bits as fb
import four_bits_portions as fp
from four_bits import BF16
from test_four_bits_gpu import decode_case

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ops():
    from lily_b200.csrc import ops as o
    return o


# few tokens and many, pages that the tcgen05 kernel takes, with one head and with two a block, and that only the mma.sync kernel takes
@pytest.mark.parametrize("nq,nkv,d,page", [(8, 2, 128, 64), (4, 4, 64, 16), (24, 2, 64, 128), (4, 1, 256, 64), (3, 1, 192, 8), (5, 1, 128, 64), (32, 4, 128, 128)])
@pytest.mark.parametrize("new,cached", [([1], [0]), ([5], [0]), ([130], [0]), ([33, 1, 200], [0, 511, 70]), ([0, 64], [40, 64]), ([300], [700]), ([700, 900], [300, 0])])
@pytest.mark.parametrize("lean", [0.0, 0.4])
def test_portions_are_as_near_as_half_precision(nq, nkv, d, page, new, cached, lean):
    lengths = [p + n for p, n in zip(cached, new)]
    _, kv, table, _ = decode_case(lengths, nq, nkv, d, page, BF16, seed=6, lean=lean)
    q = torch.randn(sum(new), nq * d, generator=torch.Generator().manual_seed(7)).to(BF16).to(DEV)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    pre = torch.tensor(cached, dtype=torch.int32, device=DEV)
    out, bound = fp.want(q, kv, table, list(zip(new, cached)), nq, nkv, d, page, d ** -0.5)
    got = ops().attention_prefill4(q, kv, table, cu, pre, cached, new, nq, nkv, d, page, d ** -0.5)
    assert fp.faults(got, out, bound) == []


@pytest.mark.parametrize("nq,nkv,d,page", [(8, 2, 128, 64), (6, 2, 128, 16), (4, 2, 192, 32)])
@pytest.mark.parametrize("power", [-100, -30, 30, 100])
def test_values_of_any_size(nq, nkv, d, page, power):
    """Values of one kv head times a power of two give its heads' outputs times it, to the bit, and the others' as they were."""
    new, cached = [260, 40], [0, 130]
    _, kv, table, _ = decode_case([p + n for p, n in zip(cached, new)], nq, nkv, d, page, BF16, seed=8, lean=0.0)
    q = torch.randn(sum(new), nq * d, generator=torch.Generator().manual_seed(9)).to(BF16).to(DEV)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    pre = torch.tensor(cached, dtype=torch.int32, device=DEV)
    run = lambda kv: ops().attention_prefill4(q, kv, table, cu, pre, cached, new, nq, nkv, d, page, d ** -0.5).view(-1, nq, d)
    want = run(kv).clone()
    moved = kv.clone()
    held = moved[:, 1, 1, page * d // 2:].contiguous().view(BF16)
    moved[:, 1, 1, page * d // 2:] = (held * 2.0 ** power).view(torch.uint8)
    got, mine = run(moved), slice(nq // nkv, 2 * nq // nkv)
    assert torch.equal(got[:, mine], want[:, mine] * 2.0 ** power)
    others = [h for h in range(nq) if h // (nq // nkv) != 1]
    assert torch.equal(got[:, others], want[:, others])


@pytest.mark.parametrize("nq,nkv,d,page,new", [(8, 2, 128, 64, 700), (4, 2, 128, 16, 90)])
def test_large_scores(nq, nkv, d, page, new):
    """Scores of up to 2^27, whose rounded products are off by several units: every row has one place's value, and none is lost to a weight above the type's largest number."""
    _, kv, table, _ = decode_case([new], nq, nkv, d, page, BF16, seed=10, lean=0.0)
    q = (torch.randn(new, nq * d, generator=torch.Generator().manual_seed(11)) * 2.0 ** 24).to(BF16).to(DEV)
    cu, pre = torch.tensor([0, new], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops().attention_prefill4(q, kv, table, cu, pre, [0], [new], nq, nkv, d, page, d ** -0.5).view(new, nq, d)
    assert bool(torch.isfinite(got).all())
    x, pages = q.double().view(new, nq, d), table[0].long()
    hidden = torch.arange(new, device=DEV)[None] > torch.arange(new, device=DEV)[:, None]
    for h in range(nq):
        k, v = (lo + s * c for c, s, lo in ([t.reshape(-1, d)[:new] for t in fb.read_rows(kv[pages, h // (nq // nkv), i], page, d, bool(i))] for i in range(2)))
        e = (x[:, h] @ k.T * d ** -0.5).masked_fill(hidden, -float("inf"))
        room = 2.0 ** -10 * d ** -0.5 * (x[:, h].abs() @ k.abs().T).amax(-1)       # (keys rounded to half precision, both of a pair)
        top = e.topk(min(2, new), -1)
        sure = (top.values[:, 0] - top.values[:, 1] > 2 * room + 30) & (torch.arange(new, device=DEV) > 0)
        assert int(sure.sum()) > new // 8
        near = (got[sure, h].double() - v[top.indices[sure, 0]]).abs() - (2.0 ** -8 + 2.0 ** -10) * v[top.indices[sure, 0]].abs()
        assert bool((near <= 1e-30).all())


@pytest.mark.parametrize("nq,nkv,d,page,new", [(8, 2, 128, 64, [300, 700, 260]), (6, 2, 128, 16, [70, 130, 9]), (4, 4, 64, 64, [900, 40, 300])])
def test_portions_that_are_shorter_on_the_device(nq, nkv, d, page, new):
    """A call that is cut for longer portions than there are, as a captured one may be when it is replayed: tiles without rows write nothing, a request without tokens takes nothing from the others, and rows
    behind the last one stay as they are."""
    for short in ([0, *new[1:]], [1, max(new[1] - 50, 2), 0], [new[0], 0, 0], [0, 0, 5]):
        cached = [0, 30, 65]
        _, kv, table, _ = decode_case([p + n for p, n in zip(cached, new)], nq, nkv, d, page, BF16, seed=12, lean=0.0)
        q = torch.randn(sum(new), nq * d, generator=torch.Generator().manual_seed(13)).to(BF16).to(DEV)
        tensors = lambda lens: (torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device=DEV), torch.tensor(cached, dtype=torch.int32, device=DEV))
        out = torch.full_like(q, 7.0)
        ops().attention_prefill4(q, kv, table, *tensors(short), cached, new, nq, nkv, d, page, d ** -0.5, out)
        torch.cuda.synchronize()
        want, bound = fp.want(q, kv, table, list(zip(short, cached)), nq, nkv, d, page, d ** -0.5)
        n = sum(short)
        assert bool(((out[:n].double() - want[:n]).abs() <= bound[:n]).all()) and bool((out[n:] == 7.0).all())
