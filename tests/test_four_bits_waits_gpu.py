"""Waits of the tcgen05 product with 4-bit weights that run out: the kernel ends, what is void is NaN, the host hears of it once, and the next call is as before."""

import pytest
import torch

import four_bits as fb
from four_bits import BF16, F32

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("m,n,k,group,zeros,out", [(17, 130, 160, 32, True, BF16), (45, 300, 2048, 64, False, F32), (128, 64, 4096, 128, True, BF16), (256, 1000, 1024, 128, False, BF16), (300, 300, 256, 64, True, F32)])
def test_a_wait_that_runs_out_makes_the_product_void_and_nothing_else(monkeypatch, m, n, k, group, zeros, out):
    """No polls at all: every block gives up with its first copies on their way (one block a tile of rows, and clusters of 2, 4 and 8)."""
    from lily_b200.csrc import ops as o
    g = torch.Generator().manual_seed(m)
    w = o.pack_weight4(*fb.make_matrix(n, k, group, zeros, g, DEV))
    x = torch.randn(m, k, generator=g).to(BF16).to(DEV)
    run = lambda: o._faces().linear4(x, *w, None, out == F32, 17, *(() if o.LINEAR4_POLLS is None else (o.LINEAR4_POLLS,)))
    first = run()
    assert bool(torch.isfinite(first).all()) and o.linear4_status() == 0
    monkeypatch.setattr(o, "LINEAR4_POLLS", 0)
    void = run()
    torch.cuda.synchronize()
    assert o.linear4_lost() >> 24 in range(1, 7) and o.linear4_lost() == 0 and o.linear4_status() == 0
    assert bool(torch.isnan(void).all())
    monkeypatch.undo()
    assert torch.equal(run(), first) and o.linear4_status() == 0


def test_a_void_call_leaves_another_call_alone(monkeypatch):
    """Nothing of a call whose waits ran out is kept: a call right behind it, that nobody asked about in between, is right."""
    from lily_b200.csrc import ops as o
    g = torch.Generator().manual_seed(0)
    w = o.pack_weight4(*fb.make_matrix(700, 2048, 64, True, g, DEV))
    x = torch.randn(100, 2048, generator=g).to(BF16).to(DEV)
    want = o.linear4(x, w)
    monkeypatch.setattr(o, "LINEAR4_POLLS", 0)
    void = o.linear4(x, w)
    monkeypatch.undo()
    after = o.linear4(x, w)
    assert torch.equal(after, want) and bool(torch.isnan(void).all()) and o.linear4_status() != 0 and o.linear4_status() == 0


def test_polls_that_are_no_number_of_them_are_refused():
    from lily_b200.csrc import ops as o
    w = o.pack_weight4(*fb.make_matrix(8, 32, 32, False, torch.Generator().manual_seed(0), DEV))
    with pytest.raises(o.KernelError, match="-1 polls"):
        o._faces().linear4(torch.zeros(20, 32, dtype=BF16, device=DEV), *w, None, False, 17, -1)
