"""Where one kernel of a 4-bit product hands over to another, without a GPU."""

import types

import pytest
import torch

from lily_b200.csrc import build, ops
from lily_b200.csrc.ops import Weight4

BF16, F32 = torch.bfloat16, torch.float32


def test_the_library_says_how_many_tokens_are_few():
    try:
        ops.library()
    except build.BuildError as exc:
        pytest.skip(f"no kernel library here: {exc}")
    assert ops.linear4_few_tokens(BF16) == 16 and ops.linear4_few_tokens(F32) == 8


@pytest.mark.parametrize("few", [1, 5, 16, 30])
def test_products_change_kernels_where_it_says(monkeypatch, few):
    """Whatever that number is: up to it the kernels for few tokens, behind it tcgen05 (bfloat16) or the matrix as numbers, and nothing in between that neither takes."""
    seen = []
    monkeypatch.setattr(ops, "linear4_few_tokens", lambda dtype: few)
    monkeypatch.setattr(ops, "_module", types.SimpleNamespace(linear4=lambda x, *a: seen.append(("few" if x.shape[0] < a[8] or x.dtype == F32 else "tcgen05", x.shape[0]))))
    monkeypatch.setattr(ops, "weights4", lambda w, dtype: "numbers")
    monkeypatch.setattr(ops, "linear", lambda x, w, *a: seen.append((w, x.shape[0])))
    w = Weight4(None, None, None, 64, 32, 32)
    for dtype, then in ((BF16, "tcgen05"), (F32, "numbers")):
        seen.clear()
        for m in (1, few, few + 1, few + 20):
            ops.linear4(torch.zeros(m, 32, dtype=dtype), w)
        assert seen == [("few", 1), ("few", few), (then, few + 1), (then, few + 20)]
