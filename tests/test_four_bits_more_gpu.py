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


@pytest.mark.parametrize("gain_dtype", [BF16, F32])
@pytest.mark.parametrize("nq,nkv,d,rot,page", [(4, 2, 128, 128, 16), (6, 2, 64, 64, 64), (2, 1, 192, 96, 16), (4, 1, 256, 256, 32), (5, 1, 128, 36, 1), (2, 2, 128, 0, 64)])
@pytest.mark.parametrize("norm", [True, False])
def test_write_of_float32_heads_with_bfloat16_queries(gain_dtype, nq, nkv, d, rot, page, norm):
    """Codes to the bit those of the plain statement on the float32 heads, queries with one rounding."""
    from test_four_bits_gpu import run_write, same_bytes, write_case, written
    c = write_case(F32, nq, nkv, d, rot, page, [3, 1, 20], [5, 70, 0], norm, gain_dtype, nq * d)
    want_q, want_kv = written(c, nq, nkv, d, rot, page, 1e-6)
    given = torch.empty(24, nq * d, dtype=BF16, device=DEV)
    q, kv = run_write(c, nq, nkv, d, rot, page, 1e-6, q_out=given)
    assert q.dtype == BF16 and torch.equal(q, want_q.to(BF16)) and torch.equal(given.cpu(), q)
    assert same_bytes(kv, want_kv, page, d)


def test_queries_of_another_type_are_refused():
    from test_four_bits_gpu import run_write, write_case
    c = write_case(BF16, 2, 1, 64, 64, 16, [3], [0], False, BF16, 1)
    with pytest.raises(ops().KernelError, match="q_out"):
        run_write(c, 2, 1, 64, 64, 16, 1e-6, q_out=torch.empty(3, 128, dtype=F32, device=DEV))
    c = write_case(F32, 2, 1, 64, 64, 16, [3], [0], False, F32, 1)
    with pytest.raises(ops().KernelError, match="q_out"):
        run_write(c, 2, 1, 64, 64, 16, 1e-6, q_out=torch.empty(3, 128, dtype=torch.float16, device=DEV))


@pytest.mark.parametrize("m", [1, 8, 16, 17])
@pytest.mark.parametrize("quantised", [True, False])
def test_heads_of_a_few_tokens_are_not_rounded_ahead_of_their_norm(m, quantised):
    """What goes into the norm and the cache: float32 sums, within 2^-18 of the magnitudes, of up to 16 tokens; bfloat16 behind that, as ever."""
    o, g, n, k = ops(), torch.Generator().manual_seed(m), 384, 256
    w = (torch.randn(n, k, generator=g) / 16).to(BF16).to(DEV)
    held = o.quantize_weight4(w, 128) if quantised else w
    full = o.weights4(held, F32).double() if quantised else w.double()
    x, bias = torch.randn(m, k, generator=g).to(BF16).to(DEV), torch.randn(n, generator=g).to(BF16).to(DEV)
    for b in (None, bias):
        got = o.linear_unrounded(x, held, b)
        assert got.dtype == (F32 if m <= 16 else BF16)
        if m <= 16:
            want = x.double() @ full.t() + (0 if b is None else b.double())
            within(got, want, 2.0 ** -18 * (x.double().abs() @ full.abs().t()) + 2.0 ** -23 * want.abs())


# ---- how decode rows are cut ----

@pytest.mark.parametrize("dtype,page", [(F32, 64), (BF16, 8)])
@pytest.mark.parametrize("nq,d,most", [(8, 256, 2), (4, 256, 3), (8, 192, 3), (8, 128, 3)])
def test_blocks_on_cuda_cores_are_no_more_than_the_device_holds(dtype, page, nq, d, most):
    """What a block has in shared memory (86,528 bytes where eight heads of 256 features are a pair, so that a multiprocessor's 233,472 hold two), looked at by the scratch that blocks leave parts in."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert ops().decode4_scratch_floats(4, nq, 1, d, 200_000, page, dtype) == 2 * most * sms * 8 * (d + 2)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq,nkv,d,page", [(16, 4, 128, 64), (8, 2, 64, 16), (8, 1, 256, 64), (6, 2, 128, 8)])
@pytest.mark.parametrize("lengths", [[1] * 8, [60] * 8, [0, 64, 0, 17], [5], [64, 3, 32], [40] * 70, [1000, 3, 90]])
def test_the_longest_row_that_may_come(dtype, nq, nkv, d, page, lengths):
    """A captured step is made for rows of thousands of places, and gives rows of any length as near as a call that is made for them."""
    q, kv, table, seq = decode_case(lengths, nq, nkv, d, page, dtype)
    run = lambda table, longest: ops().attention_decode4(q, kv, table, seq, longest, nq, nkv, d, page, d ** -0.5)
    want, by_codes, by_values = fb.attention(q, kv, table, [(1 if n else 0, n - 1 if n else 0) for n in lengths], nq, nkv, d, page, d ** -0.5)
    within(run(table, max(lengths)), want, attention_bound(by_codes, by_values, want, dtype))
    for longest in (8192, 131072):
        wide = torch.zeros(len(lengths), longest // page, dtype=torch.int32, device=DEV)
        wide[:, :table.shape[1]] = table
        got = run(wide, longest)
        within(got, want, attention_bound(by_codes, by_values, want, dtype))


@pytest.mark.parametrize("power", [60, 90, 100, 110, 118, 120, 122, 124, 125])
@pytest.mark.parametrize("nq,nkv,d,page", [(4, 1, 128, 64), (8, 2, 64, 16), (4, 1, 256, 64)])
def test_decode_of_queries_near_the_largest_numbers(nq, nkv, d, page, power):
    """Scores of up to 2^127: every head has the value of its best place, wherever that is, as far as float32 scores tell it from the next (errors of 2^-18 of sum |q_f k_f|)."""
    lengths = [900, 40, 0, 333]
    q, kv, table, seq = decode_case(lengths, nq, nkv, d, page, BF16, seed=power)
    q = (q.float().clamp(-3.9, 3.9) * 2.0 ** power).to(BF16)
    got = ops().attention_decode4(q, kv, table, seq, 900, nq, nkv, d, page, d ** -0.5).view(-1, nq, d)
    assert bool(torch.isfinite(got).all()) and bool((got[2] == 0).all())
    seen = 0
    for r, n in enumerate(lengths):
        if not n:
            continue
        pages = table[r].long()[:-(-n // page)]
        for h in range(nq):
            k, v = (lo + s * c for c, s, lo in ([t.reshape(-1, d)[:n] for t in fb.read_rows(kv[pages, h // (nq // nkv), i], page, d, bool(i))] for i in range(2)))
            x = q.view(-1, nq, d)[r, h].double()
            e, error = k @ x, 2.0 ** -18 * (k.abs() @ x.abs()).max()
            top = e.topk(2)
            if float(top.values[0] - top.values[1]) > 2 * float(error):
                seen += 1
                want = v[top.indices[0]]
                # the value through the second product: codes less the middle one, and its step, exact; the output's rounding and that of a weight of one
                within(got[r, h], want, HALF[BF16] * want.abs() + 2.0 ** -7 * want.abs() + 2.0 ** -12 * v.abs().max())
    assert seen >= nq * 3 // 2


# ---- weights times steps in half precision ----

def decode_bound(by_codes, by_values, want, largest):
    """A weight times a step rounded to half precision moves c - 8 of it (2^-11), a subnormal one (2^-24 where the largest is 2^6 or more; codes are up to 31 there, and a row's weights 2^13 at most together,
    its largest being 2^8) no more than 2^-14 of the largest value altogether; float32 sums 2^-12; the output's rounding."""
    return 2.0 ** -11 * by_codes + HALF[BF16] * want.abs() + 2.0 ** -12 * by_values + 2.0 ** -14 * largest + 1e-30


@pytest.mark.parametrize("nq,nkv,d,page", [(8, 2, 128, 64), (4, 4, 64, 16), (16, 1, 128, 16), (24, 2, 64, 128), (6, 1, 192, 32), (4, 1, 256, 64)])
@pytest.mark.parametrize("lengths", [[1], [23], [63, 64, 65], [300, 0, 1, 16, 257], [2500], [100] * 70])
def test_decode_is_as_near_as_its_outputs_rounding(nq, nkv, d, page, lengths):
    """All outputs together: no further off than the 64-bit ones' own rounding to bfloat16, r of their norm, and what weights in half precision add, 2^-11 at most and independent of it: sqrt(r^2 + 2^-22),
    a twentieth more for the rounding of numbers that are a little off.  (r itself is 1.6e-3 as a rule and is taken from the numbers: a row of one place has each of its values in all of its heads, and 128
    numbers twelve times over have r = 2.2e-3.  Weights in bfloat16 would add 1.6e-3 to long rows.)"""
    q, kv, table, seq = decode_case(lengths, nq, nkv, d, page, BF16, seed=3, lean=0.0)
    want, by_codes, by_values = fb.attention(q, kv, table, [(1 if n else 0, n - 1 if n else 0) for n in lengths], nq, nkv, d, page, d ** -0.5)
    got = ops().attention_decode4(q, kv, table, seq, max(lengths), nq, nkv, d, page, d ** -0.5)
    within(got, want, decode_bound(by_codes, by_values, want, 0.0 * want))
    r = float((want.to(BF16).double() - want).norm())
    assert float((got.double() - want).norm()) <= 1.05 * (r ** 2 + 2.0 ** -22 * float(want.norm()) ** 2) ** 0.5 + 1e-30


@pytest.mark.parametrize("nq,nkv,d,page", [(8, 2, 128, 64), (4, 4, 64, 16), (4, 1, 256, 64)])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("low,high", [(-12, 12), (-60, 60), (-110, -90), (60, 110)])
def test_decode_over_values_of_all_sizes(nq, nkv, d, page, order, low, high):
    """Values whose sizes grow along the row, so that the power of two for steps is lowered again and again, or fall, or jump: sums so far follow, and nothing overflows."""
    n = 1300
    q, kv, table, seq = decode_case([n], nq, nkv, d, page, BF16, seed=9, lean=0.0)
    power = torch.linspace(low, high, n).round()
    power = power if order == "rising" else power.flip(0) if order == "falling" else power[torch.randperm(n, generator=torch.Generator().manual_seed(1))]
    held = kv[:, :, 1, page * d // 2:].contiguous().view(BF16).view(-1, nkv, page, d // 64, 2)
    for j in range(n):
        held[table[0, j // page].long(), :, j % page] *= 2.0 ** float(power[j])
    kv[:, :, 1, page * d // 2:] = held.reshape(-1, nkv, page * d // 32).view(torch.uint8).view(-1, nkv, page * d // 16)
    want, by_codes, by_values = fb.attention(q, kv, table, [(1, n - 1)], nq, nkv, d, page, d ** -0.5)
    largest = torch.full_like(want, 0.0)
    pages = table[0].long()[:-(-n // page)]
    for kvh in range(nkv):
        c, s, lo = (t.reshape(-1, d)[:n] for t in fb.read_rows(kv[pages, kvh, 1], page, d, True))
        v = (lo + s * c).abs().amax()
        largest.view(-1, nq, d)[:, kvh * (nq // nkv):(kvh + 1) * (nq // nkv)] = v / n
    for longest in (n, 8192):
        wide = torch.zeros(1, -(-longest // page), dtype=torch.int32, device=DEV)
        wide[:, :table.shape[1]] = table
        got = ops().attention_decode4(q, kv, wide, seq, longest, nq, nkv, d, page, d ** -0.5)
        within(got, want, decode_bound(by_codes, by_values, want, largest))
