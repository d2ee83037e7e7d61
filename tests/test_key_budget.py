"""A cache held to a budget of places: the pages it gives back, and a stack of attention layers that lives on what is kept, against a
plain account of every head's keys in 64 bits.  The kernels' plain statements stand in for them on the CPU; one test runs the kernels."""

import random

import pytest
import torch

import kernel_refs
from lily_b200.bench.budget import AttentionStack, image_prompt
from lily_b200.cache.key_budget import KeyBudget
from lily_b200.cache.kv_cache import KVCacheManager
from lily_b200.cache.pages import pages_for
from lily_b200.parts.base import CacheNeed, StateNeed

CPU = torch.device("cpu")


def manager(pages=12, page=4, needs=None, device=None, states=()):
    return KVCacheManager(needs or [(CacheNeed(2, 8), 3)], list(states), page_size=page, num_pages=pages, max_requests=4, max_context=64, device=device)


# ------------------------------------------------------------------------------ pages

def test_shrink_gives_back_the_pages_behind():
    m = manager()
    s, t = m.open_request(), m.open_request()
    m.grow(s, 21)
    m.grow(t, 3)
    stamp, table = m.table_stamp(0, s), list(m.block_table(0, s))
    assert m.shrink(s, 9) == 3 and m.lengths[s] == 9 and m.block_table(0, s) == table[:3]
    assert m.table_stamp(0, s) != stamp and m.held_pages() == [4]
    stamp = m.table_stamp(0, s)
    assert m.shrink(s, 9) == 0 and m.shrink(s, 12 - 3) == 0 and m.table_stamp(0, s) == stamp       # nothing behind: the table stands
    m.grow(s, 13)
    assert len(m.block_table(0, s)) == 4 and m.block_table(0, s)[:3] == table[:3]
    assert m.shrink(s, 0) == 4 and m.block_table(0, s) == []
    m.close_request(s)
    m.close_request(t)
    assert m.held_pages() == [0] and m.free_pages() == 12


def test_shrink_refuses():
    m = manager()
    s = m.open_request()
    m.grow(s, 5)
    for n in (6, -1):
        with pytest.raises(ValueError):
            m.shrink(s, n)
    w = manager(needs=[(CacheNeed(2, 8), 1), (CacheNeed(2, 8, 6), 1)])
    s = w.open_request()
    w.grow(s, 5)
    with pytest.raises(ValueError):
        w.shrink(s, 2)
    assert w.lengths[s] == 5


@pytest.mark.parametrize("seed", range(4))
def test_growing_and_shrinking_in_any_order_keeps_the_pages_apart(seed):
    rng, m = random.Random(seed), manager(pages=20)
    for _ in range(300):
        held = list(m.lengths)
        move = rng.randrange(4)
        if move == 0 and m.slots.available:
            m.open_request()
        elif held and move == 1:
            s = rng.choice(held)
            want = min(64, m.lengths[s] + rng.randrange(9))
            if m.can_grow([(s, want)]):
                m.grow(s, want)
        elif held and move == 2:
            s = rng.choice(held)
            m.shrink(s, rng.randint(0, m.lengths[s]))
        elif held:
            m.close_request(rng.choice(held)) if rng.random() < 0.3 else None
        pages = [p for s in m.lengths for p in m.block_table(0, s)]
        assert len(set(pages)) == len(pages) == m.held_pages()[0] and 0 not in pages
        assert all(len(m.block_table(0, s)) == pages_for(n, 4) for s, n in m.lengths.items())


def test_a_budget_refuses_what_it_cannot_hold():
    for bad in (dict(keep=0), dict(keep=8, first=5, recent=4), dict(keep=8, slack=0), dict(keep=8, first=-1), dict(keep=8, recent=-1)):
        with pytest.raises(ValueError):
            KeyBudget(manager(device=CPU), ops=kernel_refs, **bad)
    with pytest.raises(ValueError):
        KeyBudget(manager(), 8, ops=kernel_refs)                                 # no device
    for need in (CacheNeed(2, 8, 6), CacheNeed(2, 8, v_head_dim=4), CacheNeed(1, 8, v_head_dim=4, values_in_keys=True)):
        with pytest.raises(ValueError):
            KeyBudget(manager(needs=[(need, 1)], device=CPU), 8, ops=kernel_refs)
    with pytest.raises(ValueError):
        KeyBudget(manager(device=CPU, states=[StateNeed((2,))]), 8, ops=kernel_refs)


def test_evict_takes_those_that_are_due_and_keeps_what_is_asked():
    m = manager(pages=16, device=CPU, needs=[(CacheNeed(2, 8), 2), (CacheNeed(1, 4), 1)])
    b = KeyBudget(m, 8, first=2, recent=3, slack=4, ops=kernel_refs)
    assert b.most == 12 and [tuple(w.shape) for w in b.weights] == [(2, 17, 2, 4), (1, 17, 1, 4)]
    slots = [m.open_request() for _ in range(3)]
    for s, n in zip(slots, (12, 11, 3)):
        m.grow(s, n)
    g = torch.Generator().manual_seed(0)
    for group, w in zip(m.groups, b.weights):
        group.data.normal_(generator=g)
        w.uniform_(generator=g)
    before = [(group.data.clone(), w.clone()) for group, w in zip(m.groups, b.weights)]
    tables = [list(m.block_table(0, s)) for s in slots]
    assert b.evict(slots) == slots[:1]
    assert [m.lengths[s] for s in slots] == [8, 11, 3] and [len(m.block_table(0, s)) for s in slots] == [2, 3, 1]
    for (data, w), group, now in zip(before, m.groups, b.weights):
        for layer, head in [(l, h) for l in range(group.num_layers) for h in range(group.need.kv_heads)]:
            flat = torch.cat([w[layer, p, head] for p in tables[0]])
            middle = sorted(range(2, 9), key=lambda i: -float(flat[i]))[:3]
            want = [0, 1] + sorted(middle) + [9, 10, 11]
            for i, j in enumerate(want):
                to, at = (tables[0][i // 4], i % 4), (tables[0][j // 4], j % 4)
                assert torch.equal(group.data[layer, to[0], :, head, to[1]], data[layer, at[0], :, head, at[1]])
                assert now[layer, to[0], head, to[1]] == w[layer, at[0], head, at[1]]
        for t in tables[1:]:
            assert torch.equal(group.data[:, t], data[:, t]) and torch.equal(now[:, t], w[:, t])
    assert b.evict(slots) == [] and b.evict(slots, force=True) == slots[1:2] and m.lengths[slots[1]] == 8


def test_image_prompt():
    p = image_prompt(2, 2, 3, 2, start=5)
    assert p.tolist() == [[5, 6, 7, 7, 7, 7, 7, 7, 10, 11], [5, 6, 7, 7, 7, 8, 8, 8, 10, 11], [5, 6, 7, 8, 9, 7, 8, 9, 10, 11]]
    assert image_prompt(3, 0, 0, 2).tolist() == [[0, 1, 2, 3, 4]] * 3
    assert p.dtype == torch.int32


# ------------------------------------------------------------------------------ a stack that lives on what is kept

class Account:
    """The stack in 64 bits with lists in place of a cache: for every layer and kv head the (key, value, weight) it still has."""

    def __init__(self, stack):
        self.s, self.kept, self.counted = stack, {}, {}

    def open(self, slot):
        self.kept[slot] = [[[] for _ in range(self.s.nkv)] for _ in range(self.s.layers)]

    def _heads(self, layer, x, at):
        s = self.s
        y = (x @ s.w_qkv[layer].double().cpu().t()).view(-1, s.nq + 2 * s.nkv, s.d)
        axis, pair = s.pair_axis.long().cpu(), torch.arange(s.d // 2)
        c, n = s.cos.double().cpu()[at[axis].t(), pair][:, None], s.sin.double().cpu()[at[axis].t(), pair][:, None]

        def turned(t, gain):
            t = t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * gain.double().cpu()
            a, b = t.chunk(2, -1)
            return torch.cat([a * c - b * n, b * c + a * n], -1)
        return turned(y[:, :s.nq], s.gain[0]), turned(y[:, s.nq:s.nq + s.nkv], s.gain[1]), y[:, s.nq + s.nkv:]

    def step(self, slot, x, at, observe=None):
        """The next tokens of one request, at positions ``at`` [3, tokens]."""
        s, x, n = self.s, x.double().cpu(), x.shape[0]
        rep = s.nq // s.nkv
        for layer in range(s.layers):
            q, k, v = self._heads(layer, x, at.long())
            out = torch.zeros(n, s.nq, s.d, dtype=torch.float64)
            for g in range(s.nkv):
                mine = self.kept[slot][layer][g]
                for t in range(n):
                    mine.append([k[t, g], v[t, g], 0.0])
                    keys, values = torch.stack([m[0] for m in mine]), torch.stack([m[1] for m in mine])
                    p = torch.softmax(q[t, g * rep:(g + 1) * rep] @ keys.t() * s.d ** -0.5, -1)
                    out[t, g * rep:(g + 1) * rep] = p @ values
                    if observe is None or t >= n - observe:
                        for m, w in zip(mine, p.sum(0).tolist()):
                            m[2] += w
            x = x + out.view(n, -1) @ s.w_o[layer].double().cpu().t()
        self._evict(slot)
        return x

    def _evict(self, slot):
        b = self.s.budget
        if b is None or len(self.kept[slot][0][0]) < b.keep + b.slack:
            return
        for heads in self.kept[slot]:
            for g, mine in enumerate(heads):
                n = len(mine)
                rest = sorted(range(b.first, n - b.recent), key=lambda i: -mine[i][2])[:b.keep - b.first - b.recent]
                heads[g] = [mine[i] for i in sorted([*range(b.first), *rest, *range(n - b.recent, n)])]


def run(stack, portions, steps, observe=None, account=True):
    """Portions of prompts, then decoded tokens, of several requests; yields (what came, what the account says)."""
    g = torch.Generator().manual_seed(7)
    book = Account(stack)
    slots = [stack.open() for _ in portions]
    for s in slots:
        book.open(s)
    rounds = max(len(p) for p in portions)
    for i in range(rounds):
        now = [(s, p[i]) for s, p in zip(slots, portions) if i < len(p)]
        xs = [torch.randn(at.shape[1], stack.w_qkv[0].shape[1], generator=g) for _, at in now]
        got = stack.portion([s for s, _ in now], [x.to(stack.device) for x in xs], [at for _, at in now], observe=observe)
        for (s, at), x, y in zip(now, xs, got):
            yield y, book.step(s, x, at, observe) if account else None
    for _ in range(steps):
        x = torch.randn(len(slots), stack.w_qkv[0].shape[1], generator=g)
        ats = [torch.full((3, 1), stack.next_position[s]) for s in slots]
        got = stack.decode(slots, x.to(stack.device))
        for i, (s, at) in enumerate(zip(slots, ats)):
            yield got[i:i + 1], book.step(s, x[i:i + 1], at) if account else None


def portions_of(kind):
    if kind == "short":
        return [[image_prompt(3, 2, 3, 2)], [image_prompt(1, 0, 0, 0)]]
    first = image_prompt(5, 3, 4, 6)                                 # 23 tokens in two portions
    return [[first[:, :13], first[:, 13:]], [image_prompt(9, 0, 0, 0)], [image_prompt(0, 4, 4, 1), image_prompt(11, 0, 0, 0, start=40)]]


def stack_of(device, dtype, ops, **kw):
    return AttentionStack(2, 24, 4, 2, 8, page_size=4, num_pages=48, max_requests=4, max_context=96, max_position=128, device=device, dtype=dtype, ops=ops, **kw)


@pytest.mark.parametrize("kind", ["short", "long"])
@pytest.mark.parametrize("budget", [dict(), dict(keep=64), dict(keep=12, first=2, recent=4, slack=1), dict(keep=10, first=0, recent=0, slack=5),
                                    dict(keep=8, first=1, recent=7, slack=3)])
@pytest.mark.parametrize("observe", [None, 3])
def test_stack_against_the_account(kind, budget, observe):
    """Float32 sums of up to 32 terms of size 1 in both: 1e-5 a sum, a handful of sums a layer."""
    stack = stack_of(CPU, torch.float32, kernel_refs, **budget)
    for got, want in run(stack, portions_of(kind), 14, observe):
        torch.testing.assert_close(got.double(), want, atol=2e-4, rtol=1e-4)
    held = list(stack.cache.lengths.values())
    if budget.get("slack"):
        assert max(held) < budget["keep"] + budget["slack"]
    for s in list(stack.cache.lengths):
        assert len(stack.cache.block_table(0, s)) == pages_for(stack.cache.lengths[s], 4)
        stack.close(s)
    assert stack.cache.held_pages() == [0]


def test_a_budget_that_nothing_reaches_changes_nothing():
    a, b = stack_of(CPU, torch.float32, kernel_refs), stack_of(CPU, torch.float32, kernel_refs, keep=80)
    for (x, _), (y, _) in zip(run(a, portions_of("long"), 5, account=False), run(b, portions_of("long"), 5, account=False)):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,d,page,layers", [(4, 2, 8, 4, 2), (8, 2, 128, 64, 2), (6, 6, 64, 16, 1)])
@pytest.mark.parametrize("budget", [dict(), dict(keep=96, first=4, recent=24, slack=8), dict(keep=150, first=0, recent=1, slack=1)])
def test_stack_of_kernels_in_float32(nq, nkv, d, page, layers, budget):
    """The kernels against the account, requests of some hundred tokens.  Sums of up to 300 terms of size 1 in float32 (2e-5 each), a handful of
    them a layer, and each layer passes its error on to the next."""
    stack = AttentionStack(layers, 64, nq, nkv, d, page_size=page, num_pages=3 * (512 // page), max_requests=3, max_context=512, max_position=512, dtype=torch.float32, **budget)
    first = image_prompt(20, 8, 9, 61)
    portions = [[first[:, :100], first[:, 100:]], [image_prompt(1, 0, 0, 0)], [image_prompt(0, 10, 12, 31)]]
    for got, want in run(stack, portions, 12):
        torch.testing.assert_close(got.double().cpu(), want, atol=1e-3, rtol=1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,d,page", [(8, 2, 128, 64), (6, 6, 64, 16), (10, 2, 40, 8)])
def test_stack_of_kernels_in_bfloat16_keeps_its_books(nq, nkv, d, page):
    """What is kept in bfloat16 may differ from the account's by a near tie, so the invariants are looked at: lengths, pages, and that the weights of
    a layer and kv head add up to the query heads that were heard, less what went with the keys that are gone."""
    stack = AttentionStack(2, 64, nq, nkv, d, page_size=page, num_pages=3 * (512 // page), max_requests=3, max_context=512, max_position=512,
                           keep=128, first=4, recent=32, slack=16)
    slots = [stack.open() for _ in range(3)]
    sizes, heard = [200, 1, 120], [0, 0, 0]
    g = torch.Generator().manual_seed(1)
    xs = [torch.randn(n, 64, generator=g).cuda() for n in sizes]
    for y in stack.portion(slots, xs, [image_prompt(n, 0, 0, 0) for n in sizes]):
        assert bool(torch.isfinite(y).all())
    assert [stack.cache.lengths[s] for s in slots] == [128, 1, 120]
    heard = list(sizes)
    for _ in range(20):
        assert bool(torch.isfinite(stack.decode(slots, torch.randn(3, 64, generator=g).cuda())).all())
        heard = [h + 1 for h in heard]
    assert [stack.cache.lengths[s] for s in slots] == [132, 21, 140]
    for s, h in zip(slots, heard):
        n, table = stack.cache.lengths[s], stack.cache.block_table(0, s)
        assert len(table) == pages_for(n, page)
        for layer in range(2):
            total = stack.budget.layer(0, layer)[table].permute(1, 0, 2).reshape(nkv, -1)[:, :n].double().sum(1).cpu()
            if h == n:                                               # nothing was evicted: the sum is every heard query head's 1
                torch.testing.assert_close(total, torch.full_like(total, h * nq / nkv), atol=0, rtol=1e-2)
            else:
                assert bool((total > 0).all()) and bool((total < h * nq / nkv).all())


def test_no_block_writes_to_a_block_that_may_not_have_started():
    """Every kernel that writes to other blocks of its cluster waits until they run, once and ahead of its first write."""
    import os
    import re

    from lily_b200.csrc import build
    found = []
    for name in ("attention_weighed.cu", "key_weights.cu", "key_weights_tcgen05.cu", "key_budget.cu", "axes_rope.cu"):
        with open(os.path.join(build.HERE, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        heads = [m.start() for m in re.finditer(r"__global__", text)] + [len(text)]
        for body in (text[a:b] for a, b in zip(heads, heads[1:])):
            write = body.find("write_to_block(")
            if write < 0:
                assert "map_shared_rank" not in body, name
                continue
            found.append(name)
            assert 0 < body.find("cluster_arrive_started();") < body.find("cluster_wait_started();") < write, name
            assert body.count("cluster_arrive_started();") == body.count("cluster_wait_started();") == 1, name
    assert found == ["attention_weighed.cu", "key_weights.cu"]


def test_faces_refuse_on_the_host():
    """What is no tensor, lies on the host, or is no number is refused with the package's error (or Python's own), not with a crash."""
    from lily_b200.csrc import build, ops
    try:
        ops.library(), ops._faces()
    except build.BuildError as exc:
        pytest.skip(f"no kernel library here: {exc}")
    t = torch.zeros(4)
    calls = [lambda x: ops.axes_rope_write(x, None, None, 1e-6, x, x, x, x, x, x, x, x, 1, 1, 4, 4, 4), lambda x: ops.attention_decode_weighed(x, x, x, x, x, 1, 1, 1, 4, 4, 0.5),
             lambda x: ops.attention_key_weights(x, x, x, x, x, x, [0], [1], 1, 1, 4, 4, 0.5), lambda x: ops.select_keys(x, x, x, 1, 1), lambda x: ops.move_keys(x, x, x, x)]
    for call in calls:
        with pytest.raises(ops.KernelError, match="CUDA device"):
            call(t)
        with pytest.raises(ops.KernelError, match="take tensors, got int"):
            call(3)
    floats = lambda *a, **k: ops.key_weights_scratch_floats(*a, 16, 4, 128, 16, 0.1, torch.float32, **k)
    assert floats([0, 300], [333, 70]) > floats([0], [333]) > floats([0], [0]) == 0
    for bad in (([0], [-1]), ([-1], [1]), ([0], [1, 2])):
        with pytest.raises(ops.KernelError):
            floats(*bad)
    for bad in (([0], 3), ([0], ["a"])):
        with pytest.raises(TypeError):
            floats(*bad)
    with pytest.raises(ops.KernelError, match="heard"):
        floats([0], [1], observe=0)
    with pytest.raises(ops.KernelError, match="32-bit"):
        floats([0], [1 << 40])
