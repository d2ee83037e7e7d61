"""More of serving in four bits: matrices of many rows, how decode rows are cut, float32 sums that the engine hands on."""

import pytest
import torch

import four_bits as fb
from four_bits import BF16, F32, HALF
from test_four_bits_gpu import attention_bound, decode_case, within

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ops():
    from lily_b200.csrc import ops as o
    return o


@pytest.mark.parametrize("dtype,m", [(BF16, 4), (BF16, 300), (BF16, 600), (F32, 3), (F32, 12)])
def test_more_rows_than_a_launch_takes(dtype, m):
    """A matrix of more than 65,535 x 8 rows, whatever the number of tokens and so the kernel: its first rows, those on both sides of that number, its last."""
    n, k = 65535 * 8 + 77, 32
    g = torch.Generator(device=DEV).manual_seed(m)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8, device=DEV)
    scales = (torch.rand(n, 1, generator=g, device=DEV) + 0.1).to(BF16)
    w4 = ops().pack_weight4(codes, scales)
    x = torch.randn(m, k, generator=g, device=DEV).to(dtype)
    rows = torch.cat([torch.arange(40), torch.arange(65535 * 8 - 40, n)]).to(DEV)
    w = fb.matrix_values(codes[rows], scales[rows], None)
    assert torch.equal(ops().weights4(w4, dtype)[rows], w.to(dtype))
    got, want = ops().linear4(x, w4)[:, rows], x.double() @ w.t()
    size = x.double().abs() @ w.abs().t()
    within(got, want, 2.0 ** -18 * size + HALF[dtype] * want.abs() + (HALF[BF16] * size if dtype == BF16 and m > 16 else 0))


# ---- what the engine hands on ----

@pytest.mark.parametrize("m", [1, 8, 16])
@pytest.mark.parametrize("group", [32, 128])
def test_a_few_tokens_gate_is_rounded_once(m, group):
    """A gated feed-forward's first half with its matrices in four bits: sums of gate and up reach the activation in float32, as they do without four bits."""
    from lily_b200.parts.base import BuildContext
    from lily_b200.parts.mlp import SwiGLU, SwiGLUSpec
    o, g, hidden, inner = ops(), torch.Generator().manual_seed(m), 256, 384
    part = SwiGLU(SwiGLUSpec(hidden, inner), "m", BuildContext(torch.device(DEV), BF16, o, weight_group=group))
    made = {name: (torch.randn(spec.shape, generator=g) / 16).to(BF16).to(DEV) for name, spec in part.tensors().items()}
    part.load(lambda name: made[name])
    x = torch.randn(m, hidden, generator=g).to(BF16).to(DEV)
    sums = o.linear_auto(x, part.w_gate_up)
    assert sums.dtype == F32 and sums.shape == (1, m, 2 * inner)
    got = o.silu_mul(sums, BF16).double()
    w = o.weights4(part.w_gate_up, F32).double()
    y, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    gate, up = y.split(inner, 1)
    want = gate * torch.sigmoid(gate) * up
    # float32 sums (2^-18 of the magnitudes, as in test_product), whose errors the gate passes on at a slope of 1.1 at most; exponential and quotient 2^-20; one rounding
    moved = 2.0 ** -18 * (1.1 * size[:, :inner] * up.abs() + gate.abs() * size[:, inner:]) + 2.0 ** -20 * want.abs()
    within(got, want, moved + HALF[BF16] * (want.abs() + moved))
    # the whole part: the same activation through the second matrix, float32 sums too
    down, act = o.weights4(part.w_down, F32).double(), o.silu_mul(sums, BF16)
    out = part.forward(x, None)
    assert out.dtype == F32
    within(out.sum(0) if out.dim() == 3 else out, act.double() @ down.t(), 2.0 ** -18 * (act.double().abs() @ down.abs().t()))
