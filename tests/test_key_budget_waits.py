"""What a budget of cached keys looks at before it lets go of anything: waits that kernels gave up, requests that are named twice."""

import types

import pytest
import torch

import kernel_refs
from lily_b200.bench.budget import AttentionStack, image_prompt
from lily_b200.cache.key_budget import KeyBudget
from lily_b200.cache.kv_cache import KVCacheManager
from lily_b200.csrc import waits
from lily_b200.parts.base import CacheNeed


def reporting(decode=(), weights=()):
    """The kernels' plain statements, whose words say these things in turn, then nothing."""
    decode, weights = iter(decode), iter(weights)
    return types.SimpleNamespace(**{k: v for k, v in vars(kernel_refs).items() if not k.startswith("__")}, attention_decode_lost=lambda: next(decode, 0),
                                 key_weights_lost=lambda: next(weights, 0))


def full(ops, **kw):
    cache = KVCacheManager([(CacheNeed(2, 8), 2)], [], page_size=4, num_pages=16, max_requests=4, max_context=64, device=torch.device("cpu"))
    budget = KeyBudget(cache, 8, first=2, recent=3, slack=4, ops=ops, **kw)
    slot = cache.open_request()
    cache.grow(slot, 13)
    g = torch.Generator().manual_seed(0)
    cache.groups[0].data.normal_(generator=g)
    budget.weights[0].uniform_(generator=g)
    return cache, budget, slot


@pytest.mark.parametrize("words,said", [(dict(decode=[5]), "row 4 of its step"), (dict(weights=[7 << 24 | 31]), "code 7, block 31"), (dict(decode=[2], weights=[1 << 24]), "row 1 of its step")])
def test_nothing_is_let_go_of_where_a_wait_was_given_up(words, said):
    cache, budget, slot = full(reporting(**words))
    data, w, pages = cache.groups[0].data.clone(), budget.weights[0].clone(), list(cache.block_table(0, slot))
    with pytest.raises(RuntimeError, match=said):
        budget.evict([slot])
    assert torch.equal(cache.groups[0].data, data) and torch.equal(budget.weights[0], w) and cache.block_table(0, slot) == pages and cache.lengths[slot] == 13
    assert budget.evict([slot]) == [slot] and cache.lengths[slot] == 8          # heard once


def test_a_request_that_is_named_twice_is_evicted_once(monkeypatch):
    """Two lists of one request would be moved in place at the same time."""
    ops = reporting()
    cache, budget, slot = full(ops)
    asked = []
    monkeypatch.setattr(ops, "move_keys", lambda kv, w, table, kept: asked.append(table.shape[0]))
    assert budget.evict([slot, slot]) == [slot] and asked == [1] and cache.lengths[slot] == 8


def test_a_request_within_its_budget_asks_for_nothing():
    cache, budget, slot = full(reporting(decode=[5]))
    cache.shrink(slot, 11)
    assert budget.evict([slot]) == []
    with pytest.raises(RuntimeError):
        budget.check_waits()


def test_every_budget_hears_of_each_and_a_later_one_of_none():
    ops = reporting(weights=[0, 3 << 24])
    one, other = full(ops)[1], full(ops)[1]
    one.check_waits()
    for b in (other, one):
        with pytest.raises(RuntimeError, match="code 3"):
            b.check_waits()
        b.check_waits()
    full(ops)[1].check_waits()
    assert waits.KEY_WEIGHTS.row == 3 << 24


@pytest.mark.gpu
@pytest.mark.parametrize("limit,when", [("KEY_WEIGHTS_POLLS", "portion"), ("DECODE_POLLS", "decode")])
def test_a_stack_whose_kernels_give_up_lets_go_of_no_key(monkeypatch, limit, when):
    """The word is there when the eviction looks, although nobody has waited for the step."""
    from lily_b200.csrc import ops
    stack = AttentionStack(2, 64, 8, 2, 128, page_size=64, num_pages=32, max_requests=2, max_context=1024, max_position=1024, keep=128, first=4, recent=32, slack=2)
    slots = [stack.open() for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = lambda n: [torch.randn(n, 64, device="cuda", generator=g) for _ in slots]
    step = (lambda: stack.portion(slots, rows(200), [image_prompt(200, 0, 0, 0, start=stack.next_position[s]) for s in slots])) if when == "portion" else \
        (lambda: stack.decode(slots, torch.cat(rows(1))))
    stack.portion(slots, rows(129), [image_prompt(129, 0, 0, 0) for _ in slots])
    held = [stack.cache.lengths[s] for s in slots]
    monkeypatch.setattr(ops, limit, (0, 0) if when == "portion" else 0)
    with pytest.raises(RuntimeError, match="void"):
        step()
    assert [stack.cache.lengths[s] for s in slots] == [h + (200 if when == "portion" else 1) for h in held]
    monkeypatch.undo()
    stack.check_waits()
    step()
    assert [stack.cache.lengths[s] for s in slots] == [128, 128]
    torch.cuda.synchronize()
    stack.check_waits()
