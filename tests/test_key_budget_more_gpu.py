"""More of a cache held to a budget, on the GPU: waits that run out, calls of many requests, portions without tokens, ranges two blocks share, and
steps captured in a graph."""

import pytest
import torch

import test_key_budget_gpu as base
from test_key_budget_gpu import BF16, DEV, F32, close, decode_want, pool, portion_want, same

pytestmark = pytest.mark.gpu


def ops():
    from lily_b200.csrc import ops as o
    return o


@pytest.mark.parametrize("lengths,nq,nkv,d", [([70], 4, 2, 128), ([900, 33, 0, 1200], 16, 4, 128), ([900, 33, 0, 1200], 16, 4, 64), ([500] * 150, 16, 4, 64), ([20000, 400], 8, 1, 128)])
def test_a_wait_that_runs_out_is_reported_and_the_next_step_is_as_before(monkeypatch, lengths, nq, nkv, d):
    """Pages of 64: tiles by TMA.  One block a row, clusters, ranges that a second kernel joins."""
    o, page = ops(), 64
    kv, w, table = pool(lengths, nkv, page, d, BF16, 3)
    q = torch.randn(len(lengths), nq * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(BF16)
    seq = torch.tensor(lengths, dtype=torch.int32, device=DEV)

    def run():
        mine = w.clone()
        out = o.attention_decode_weighed(q, kv, mine, table, seq, max(lengths), nq, nkv, d, page, d ** -0.5)
        torch.cuda.synchronize()
        return out, mine
    out, given = run()
    assert o.attention_decode_lost() == 0
    monkeypatch.setattr(o, "DECODE_POLLS", 0)
    lost, _ = run()
    some = seq > 0
    assert bool(torch.isnan(lost[some]).all()) and not bool(lost[~some].any())
    assert 1 <= o.attention_decode_lost() <= len(lengths) and o.attention_decode_lost() == 0
    monkeypatch.undo()
    again, given_again = run()
    assert torch.equal(again, out) and same(given_again, given) and o.attention_decode_lost() == 0


@pytest.mark.parametrize("d", [64, 128])
def test_two_blocks_a_pair_where_rows_are_long_and_a_little_too_many(d):
    nq, nkv, page = 16, 8, 64
    lengths = [1 + (i * 37) % 200 for i in range(59)] + [4200]
    kv, w, table = pool(lengths, nkv, page, d, BF16, 5)
    q = torch.randn(len(lengths), nq * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(BF16)
    want, want_w = decode_want(q, kv, w, table, lengths, nq, nkv, d, page, d ** -0.5)
    got = ops().attention_decode_weighed(q, kv, w, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), 4200, nq, nkv, d, page, d ** -0.5)
    close(got, want, BF16)
    close(w, want_w, F32)


@pytest.mark.parametrize("dtype,d,page", [(F32, 40, 4), (F32, 64, 16), (BF16, 64, 16), (BF16, 128, 64), (BF16, 48, 8)])
@pytest.mark.parametrize("requests", [41, 97])
def test_portions_of_many_requests_in_one_call(dtype, d, page, requests):
    """More requests than a launch describes; every fifth brings no token."""
    nq, nkv = 4, 2
    new = [0 if r % 5 == 3 else 1 + (r * 11) % 23 for r in range(requests)]
    cached = [(r * 29) % 40 for r in range(requests)]
    kv, w, table = pool([c + n for c, n in zip(cached, new)], nkv, page, d, dtype, 9)
    q = torch.randn(sum(new), nq * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).to(dtype)
    want = portion_want(q, kv, w, table, cached, new, nq, nkv, d, page, d ** -0.5, None)
    cu = torch.tensor([sum(new[:r]) for r in range(requests + 1)], dtype=torch.int32, device=DEV)
    ops().attention_key_weights(q, kv, w, table, cu, torch.tensor(cached, dtype=torch.int32, device=DEV), cached, new, nq, nkv, d, page, d ** -0.5)
    close(w, want, F32)
    assert ops().key_weights_status() == 0


def test_no_tokens_at_all_change_nothing():
    kv, w, table = pool([30, 7], 2, 16, 64, BF16, 1)
    before = w.clone()
    zero = torch.zeros(3, dtype=torch.int32, device=DEV)
    ops().attention_key_weights(torch.zeros(0, 4 * 64, dtype=BF16, device=DEV), kv, w, table, zero, torch.tensor([30, 7], dtype=torch.int32, device=DEV), [30, 7], [0, 0], 4, 2, 64, 16, 0.1)
    q = ops().axes_rope_write(torch.zeros(0, 8 * 64, dtype=BF16, device=DEV), None, None, 1e-6, torch.ones(4, 32, device=DEV), torch.ones(4, 32, device=DEV), zero[None, :0].contiguous(),
                              ops().pair_axes((32,), DEV), zero[:0], zero[:0], table, kv, 4, 2, 64, 64, 16)
    assert q.shape == (0, 256) and same(w, before)


def test_a_captured_step_runs_again_on_what_has_changed():
    """Rotation and write, attention, selection and move in one graph: replayed, it does what the calls do."""
    o, nq, nkv, d, page, n = ops(), 8, 2, 128, 64, 200
    g = torch.Generator(device=DEV).manual_seed(4)
    kv, w, table = pool([n, n], nkv, page, d, BF16, 2)
    angle = torch.rand(300, d // 2, device=DEV, generator=g)
    qkv = torch.randn(2, (nq + 2 * nkv) * d, device=DEV, generator=g).to(BF16)
    at = torch.full((3, 2), 250, dtype=torch.int32, device=DEV)
    places, req, seq = torch.full((2,), n - 1, dtype=torch.int32, device=DEV), torch.arange(2, dtype=torch.int32, device=DEV), torch.full((2,), n, dtype=torch.int32, device=DEV)
    axes = o.pair_axes((16, 24, 24), DEV)

    def step(kv, w):
        q = o.axes_rope_write(qkv, None, None, 1e-6, angle.cos(), angle.sin(), at, axes, places, req, table, kv, nq, nkv, d, d, page)
        out = o.attention_decode_weighed(q, kv, w, table, seq, n, nq, nkv, d, page, d ** -0.5)
        o.move_keys(kv, w, table, o.select_keys(w, table, seq, n, 96, 4, 20))
        return out
    mine, given = kv.clone(), w.clone()
    step(mine.clone(), given.clone())                              # everything that is set up once
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(mine, given)
    for seed in (5, 6):
        qkv.copy_(torch.randn(qkv.shape, device=DEV, generator=g).to(BF16))
        mine.copy_(kv)
        given.copy_(w)
        graph.replay()
        other, other_w = kv.clone(), w.clone()
        want = step(other, other_w)
        assert torch.equal(out, want) and same(mine, other) and same(given, other_w)


@pytest.mark.parametrize("dtype,d,page", [(F32, 128, 16), (F32, 40, 2), (BF16, 128, 64), (BF16, 64, 16), (BF16, 24, 8)])
@pytest.mark.parametrize("rows,longest", [(1, 0), (3, 0), (3, 5), (1, 1)])
def test_rows_without_places(dtype, d, page, rows, longest):
    """All rows empty (a plan for none, or for some), and a single place."""
    lengths = [longest if longest == 1 else 0] * rows
    kv, w, table = pool([max(1, longest)] * rows, 2, page, d, dtype, 3)
    q = torch.randn(rows, 4 * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype)
    want, want_w = decode_want(q, kv, w, table, lengths, 4, 2, d, page, 0.2)
    got = ops().attention_decode_weighed(q, kv, w, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), longest, 4, 2, d, page, 0.2)
    close(got, want, dtype)
    close(w, want_w, F32)
    kept = ops().select_keys(w, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), longest, 4, 1, 1)
    assert kept.shape == (1, rows, 2, 4) and kept[..., 0].tolist() == [[[lengths[0] - 1] * 2] * rows] and bool((kept[..., 1:] == -1).all())


@pytest.mark.parametrize("n,keep,first,recent", [(3000, 512, 4, 64), (8192, 100, 0, 0), (8193, 8192, 1, 8191), (60000, 1024, 4, 128), (4097, 4096, 0, 1), (33, 32, 0, 0)])
@pytest.mark.parametrize("kind", ["few values", "all alike", "negative and infinite", "neighbours"])
def test_selection_of_equal_and_close_weights(n, keep, first, recent, kind):
    """Ties go to the lower place, however many share a weight; weights that differ in their last bits alone."""
    nkv, page = 2, 64
    g = torch.Generator().manual_seed(n)
    _, w, table = pool([n], nkv, page, 4, F32, 6)
    rows = {"few values": torch.randint(0, 5, (nkv, n), generator=g).float(), "all alike": torch.full((nkv, n), 0.25), "neighbours": (1.0 + torch.randint(0, 40, (nkv, n), generator=g) * 2.0 ** -23),
            "negative and infinite": torch.where(torch.rand(nkv, n, generator=g) < 0.01, torch.tensor(float("inf")), torch.randn(nkv, n, generator=g))}[kind]
    base.put_rows(w, table, 0, rows.to(DEV), page)
    kept = ops().select_keys(w, table, torch.tensor([n], dtype=torch.int32, device=DEV), n, keep, first, recent)[0, 0].cpu()
    for h in range(nkv):
        order = sorted(range(first, n - recent), key=lambda j: (-float(rows[h, j]), j))[:keep - first - recent]
        assert kept[h].tolist() == sorted([*range(first), *order, *range(n - recent, n)])
