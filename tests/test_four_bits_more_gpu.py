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
