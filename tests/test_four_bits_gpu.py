"""The kernels of serving in four bits, each against its definition in 64 bits: products with 4-bit weights, norm + rotation + write into a 4-bit cache, attention of
one token a request and of prompt portions over it.  Pages are shuffled, and nothing outside a call's places changes."""

import math

import pytest
import torch

import four_bits as fb
from four_bits import BF16, F32, HALF

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ops():
    from lily_b200.csrc import ops as o
    return o


def within(got, want, bound):
    """Every number no further from ``want`` than ``bound``; NaN where NaN is wanted."""
    got, want, bound = got.double(), want.double(), bound.double()
    assert got.shape == want.shape
    assert bool((torch.isnan(got) == torch.isnan(want)).all()), "NaN in other places"
    over = ((got - want).abs() - bound).nan_to_num(nan=-1.0)
    assert bool((over <= 0).all()), f"{int((over > 0).sum())} of {over.numel()} beyond their bound, by up to {float(over.max()):.3g} (bound there {float(bound.flatten()[over.argmax()]):.3g})"


# ---- products ----

def product_bound(x, w, y, dtype, out_dtype, rounded_weights):
    """float32 sums of products (2^-24 a rounding and some sixteen of them on any path of additions, the tensor cores' cut ones twice that: 2^-18 of the sum of magnitudes), one rounding of the result,
    and of each weight where more tokens than a few are taken in bfloat16."""
    size = x.double().abs() @ w.abs().t()
    return 2.0 ** -18 * size + HALF[out_dtype] * y.abs() + (HALF[BF16] * size if rounded_weights else 0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m", [1, 3, 8, 9, 16, 17, 45, 130, 300])
@pytest.mark.parametrize("n,k,group,zeros", [(128, 128, 128, False), (1, 32, 32, True), (200, 192, 64, False), (33, 1120, 32, True), (1000, 2048, 128, True), (513, 4160, 64, False)])
def test_product(dtype, m, n, k, group, zeros):
    g = torch.Generator().manual_seed(m * 7 + n)
    codes, scales, z = fb.make_matrix(n, k, group, zeros, g, DEV)
    x = torch.randn(m, k, generator=g).to(dtype).to(DEV)
    w = fb.matrix_values(codes, scales, z)
    want = x.double() @ w.t()
    got = ops().linear4(x, ops().pack_weight4(codes, scales, z))
    assert got.dtype == dtype and got.shape == (m, n)
    within(got, want, product_bound(x, w, want, dtype, dtype, dtype == BF16 and m > 16))


@pytest.mark.parametrize("m,out", [(300, BF16), (300, F32), (600, BF16), (600, F32)])
@pytest.mark.parametrize("bias_dtype", [BF16, F32])
def test_many_tokens_with_bias_and_wide_result(m, out, bias_dtype):
    """Through numbers in memory, by ``linear4`` and by ``linear``."""
    g = torch.Generator().manual_seed(m)
    codes, scales, z = fb.make_matrix(300, 256, 64, True, g, DEV)
    x, bias = torch.randn(m, 256, generator=g).to(BF16).to(DEV), torch.randn(300, generator=g).to(bias_dtype).to(DEV)
    w, w4 = fb.matrix_values(codes, scales, z), ops().pack_weight4(codes, scales, z)
    want = x.double() @ w.t() + bias.double()
    for product in (ops().linear4, ops().linear):
        got = product(x, w4, bias, out_dtype=out)
        assert got.dtype == out
        # (the library may round sums to bfloat16 ahead of the bias: one rounding more)
        within(got, want, product_bound(x, w, want, BF16, out, True) + HALF[BF16] * ((want - bias.double()).abs() + bias.double().abs()))


@pytest.mark.parametrize("m", [17, 65, 128, 129, 256, 257, 300, 600])
@pytest.mark.parametrize("n,k,group,zeros", [(130, 160, 32, True), (300, 1088, 64, False), (64, 4096, 128, True)])
def test_product_on_the_way(m, n, k, group, zeros):
    """The tcgen05 kernel itself, whichever side of the line sizes are."""
    g = torch.Generator().manual_seed(m + n)
    codes, scales, z = fb.make_matrix(n, k, group, zeros, g, DEV)
    x = torch.randn(m, k, generator=g).to(BF16).to(DEV)
    w = fb.matrix_values(codes, scales, z)
    want = x.double() @ w.t()
    got = ops()._faces().linear4(x, *ops().pack_weight4(codes, scales, z), None, False, 17)
    within(got, want, product_bound(x, w, want, BF16, BF16, True))
    assert ops().linear4_status() == 0


@pytest.mark.parametrize("dtype,m,out", [(BF16, 5, BF16), (BF16, 5, F32), (BF16, 40, BF16), (BF16, 40, F32), (F32, 5, F32), (F32, 40, F32)])
@pytest.mark.parametrize("bias_dtype", [None, BF16, F32])
def test_product_with_bias_and_wide_result(dtype, m, out, bias_dtype):
    if dtype == F32 and bias_dtype == BF16:
        return
    g = torch.Generator().manual_seed(3)
    codes, scales, z = fb.make_matrix(300, 256, 64, True, g, DEV)
    x = torch.randn(m, 256, generator=g).to(dtype).to(DEV)
    bias = None if bias_dtype is None else torch.randn(300, generator=g).to(bias_dtype).to(DEV)
    w = fb.matrix_values(codes, scales, z)
    want = x.double() @ w.t() + (0 if bias is None else bias.double())
    got = ops().linear4(x, ops().pack_weight4(codes, scales, z), bias, out_dtype=out)
    assert got.dtype == out
    extra = 0 if bias is None else 2 * HALF[BF16 if out == BF16 else F32] * bias.double().abs()
    within(got, want, product_bound(x, w, want, dtype, out, dtype == BF16 and m > 16) + extra)


@pytest.mark.parametrize("m", [2, 20])
def test_product_rows_are_their_own(m):
    """A token without a number, or with an infinite one, spoils its own row; what lies behind the last row and column is not looked at."""
    o, g = ops(), torch.Generator().manual_seed(1)
    codes, scales, z = fb.make_matrix(130, 160, 32, True, g, DEV)
    w4 = o.pack_weight4(codes, scales, z)
    full = w4.scales.transpose(1, 2).reshape(256, -1)                    # [rows, groups]
    full[130:] = math.nan
    full[:, 5:] = math.nan
    w4 = w4._replace(scales=full.view(2, 128, -1).transpose(1, 2).contiguous())
    x = torch.randn(m, 160, generator=g).to(BF16).to(DEV)
    clean = o.linear4(x, w4)
    assert bool(torch.isfinite(clean).all())
    x[1, 7] = math.nan
    got = o.linear4(x, w4)
    keep = torch.arange(m, device=DEV) != 1
    assert torch.equal(got[keep], clean[keep]) and bool(torch.isnan(got[1]).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,k,group,zeros", [(7, 32, 32, True), (300, 1120, 32, False), (128, 640, 128, True)])
def test_weights_as_numbers(dtype, n, k, group, zeros):
    g = torch.Generator().manual_seed(2)
    codes, scales, z = fb.make_matrix(n, k, group, zeros, g, DEV)
    assert torch.equal(ops().weights4(ops().pack_weight4(codes, scales, z), dtype), fb.matrix_values(codes, scales, z).to(dtype))


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantized_matrix_is_near(zeros, group):
    """No number is further off than half a scale (a rounding of the scale to bfloat16 moves the outer codes by up to 8 and 15 times 2^-8 of a scale more; the largest positive one of a group
    around 8 is kept at 15, another half of a scale off)."""
    g = torch.Generator().manual_seed(4)
    w = torch.randn(70, 384, generator=g).to(DEV) + 0.3
    q = ops().quantize_weight4(w, group, zeros)
    scales = q.scales.transpose(1, 2).reshape(128, -1)[:70, :384 // group].double().repeat_interleave(group, 1)
    off = (ops().weights4(q).double() - w.double()).abs() / scales
    assert float(off.max()) <= (0.5 + 15 / 256 + 0.5 if zeros else 1.0 + 8 / 256)
    assert float(off.mean()) < 0.3


# ---- the cache ----

def write_case(dtype, nq, nkv, d, rot, page, news, cached, norm, gain_dtype, seed, kv=None):
    g = torch.Generator().manual_seed(seed)
    n = sum(news)
    table, pages = fb.tables([c + t for c, t in zip(cached, news)], page, g)
    if kv is None:
        kv = fb.random_cache(pages, nkv, page, d, g)
    qkv = torch.randn(n, (nq + 2 * nkv) * d, generator=g).to(dtype)
    gains = [(1 + 0.2 * torch.randn(d, generator=g)).to(gain_dtype) for _ in range(2)] if norm else [None, None]
    angle = torch.outer(torch.arange(300.0), 1.0 / 100.0 ** (torch.arange(0, max(rot, 1), 2) / max(rot, 1)))[:, :rot // 2].contiguous()
    positions = torch.cat([c + torch.arange(t) for c, t in zip(cached, news)]).int()
    req = torch.repeat_interleave(torch.arange(len(news)), torch.tensor(news)).int()
    return dict(qkv=qkv, gains=gains, cos=angle.cos(), sin=angle.sin(), positions=positions, req=req, table=table, kv=kv)


def written(c, nq, nkv, d, rot, page, eps):
    """(q, cache) after the call, one IEEE operation after the other on the CPU."""
    x = c["qkv"].float().view(-1, nq + 2 * nkv, d)
    at = c["positions"].long()
    known = at < c["cos"].shape[0]
    cos, sin = (torch.where(known[:, None], t[at.clamp(max=t.shape[0] - 1)], math.nan) for t in (c["cos"], c["sin"]))
    q = fb.turn(x[:, :nq], c["gains"][0], eps, cos, sin, rot)
    k, v = fb.turn(x[:, nq:nq + nkv], c["gains"][1], eps, cos, sin, rot), x[:, nq + nkv:]
    kv = c["kv"].clone()
    for value, heads in enumerate((k, v)):
        codes, held = fb.hold(heads)
        for t, (r, p) in enumerate(zip(c["req"].tolist(), at.tolist())):
            if 0 <= r < c["table"].shape[0] and p // page < c["table"].shape[1] and 0 <= c["table"][r, p // page] < kv.shape[0]:
                for h in range(nkv):
                    fb.write_row(kv[c["table"][r, p // page], h, value], p % page, page, d, bool(value), codes[t, h], held[t, h])
    return q.reshape(len(x), nq * d), kv


def run_write(c, nq, nkv, d, rot, page, eps, **kw):
    dev = {k: v.to(DEV) for k, v in c.items() if isinstance(v, torch.Tensor)}
    gains = [None if t is None else t.to(DEV) for t in c["gains"]]
    q = ops().qk_norm_rope_write4(dev["qkv"], *gains, eps, dev["cos"], dev["sin"], dev["positions"], dev["req"], dev["table"], dev["kv"], nq, nkv, d, rot, page, **kw)
    return q.cpu(), dev["kv"].cpu()


def same_bytes(got, want, page, d):
    """Equal bytes, but for how a NaN is written."""
    if torch.equal(got, want):
        return True
    codes = page * d // 2
    a, b = (t[..., codes:].contiguous().view(BF16) for t in (got, want))
    return torch.equal(got[..., :codes], want[..., :codes]) and bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


@pytest.mark.parametrize("dtype,gain_dtype", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("nq,nkv,d,rot,page", [(4, 2, 128, 128, 16), (6, 2, 64, 64, 64), (3, 3, 64, 32, 8), (2, 1, 192, 96, 16), (4, 1, 256, 256, 32), (5, 1, 128, 36, 1), (2, 2, 128, 0, 64)])
@pytest.mark.parametrize("norm", [True, False])
def test_write(dtype, gain_dtype, nq, nkv, d, rot, page, norm):
    """The same codes as the plain statement's, to the bit; queries with one rounding; nothing else in the cache changes."""
    c = write_case(dtype, nq, nkv, d, rot, page, [3, 1, 20], [5, 70, 0], norm, gain_dtype, nq * d)
    want_q, want_kv = written(c, nq, nkv, d, rot, page, 1e-6)
    q, kv = run_write(c, nq, nkv, d, rot, page, 1e-6)
    assert q.dtype == dtype and torch.equal(q, want_q.to(dtype))
    assert same_bytes(kv, want_kv, page, d)


def test_a_token_has_the_same_codes_alone_and_in_a_prompt():
    nq, nkv, d, page = 8, 2, 128, 16
    c = write_case(BF16, nq, nkv, d, d, page, [40], [0], True, BF16, 9)
    _, whole = run_write(c, nq, nkv, d, d, page, 1e-5)
    for t in range(40):
        one = dict(c, qkv=c["qkv"][t:t + 1].clone(), positions=c["positions"][t:t + 1], req=c["req"][t:t + 1])
        _, c["kv"] = run_write(one, nq, nkv, d, d, page, 1e-5)
    assert torch.equal(c["kv"], whole)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_write_of_what_is_no_number(dtype):
    """Equal numbers, zeros, tiny ones, huge ones, infinities and NaN; a group that is not finite reads as NaN, its neighbours as ever."""
    nq, nkv, d, page = 1, 2, 128, 8
    c = write_case(dtype, nq, nkv, d, 0, page, [9], [3], False, dtype, 5)
    x = c["qkv"].view(9, nq + 2 * nkv, d)
    x[0] = 0.0
    x[1] = -3.0
    x[2, :, 64:] = 1e-30 * torch.randn(64)
    x[3, :, 5] = math.nan
    x[4, :, 70] = math.inf
    x[5, :, 3] = -math.inf
    x[6] *= 1e38
    x[7] = 1e-42
    x[8, :, :2] = torch.tensor([3e38, -3e38])
    want_q, want_kv = written(c, nq, nkv, d, 0, page, 1e-6)
    q, kv = run_write(c, nq, nkv, d, 0, page, 1e-6)
    assert torch.equal(q.nan_to_num(nan=123.0), want_q.to(dtype).nan_to_num(nan=123.0))
    assert same_bytes(kv, want_kv, page, d)
    values = ops().cache4_values(kv.to(DEV), c["table"].to(DEV), nkv, d, page, F32)[0].cpu().permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, 3:12]      # [2, nkv, tokens, d]
    nan = torch.isnan(values)
    assert bool(nan[:, :, 3, :64].all()) and not bool(nan[:, :, 3, 64:].any()) and bool(nan[:, :, 4, 64:].all()) and not bool(nan[:, :, 4, :64].any())
    assert bool((values[:, :, 1] == -3.0).all()) and bool((values[:, :, 0] == 0.0).all())


def test_write_outside_the_tables():
    """Requests, positions and pages outside their tables are not written, a position outside the rotation tables gives NaN."""
    nq, nkv, d, page = 2, 1, 64, 16
    c = write_case(F32, nq, nkv, d, d, page, [4, 4], [0, 296], False, F32, 6)       # (positions 296 to 299 of 300)
    c["req"] = torch.tensor([0, 7, -1, 0, 1, 1, 1, 1], dtype=torch.int32)
    c["positions"] = torch.tensor([0, 1, 2, 3, 296, 400, 299, -1], dtype=torch.int32)
    c["table"][0, 0] = 10000
    base = c["kv"].clone()
    q, kv = run_write(c, nq, nkv, d, d, page, 1e-6)
    assert bool(torch.isnan(q[5]).all()) and bool(torch.isnan(q[7]).all()) and bool(torch.isfinite(q[[0, 1, 2, 3, 4, 6]]).all())
    c["positions"][7], c["req"][7] = 0, 9
    want = written(dict(c, kv=base, req=torch.tensor([0, 7, 9, 0, 1, 9, 1, 9], dtype=torch.int32)), nq, nkv, d, d, page, 1e-6)[1]
    assert same_bytes(kv, want, page, d)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nkv,d,page", [(1, 64, 1), (3, 128, 64), (2, 192, 16), (1, 256, 128)])
def test_values(dtype, nkv, d, page):
    g = torch.Generator().manual_seed(8)
    kv = fb.random_cache(7, nkv, page, d, g)
    table = torch.tensor([[3, 1, 900], [6, -5, 2]], dtype=torch.int32)
    got = ops().cache4_values(kv.to(DEV), table.to(DEV), nkv, d, page, dtype).cpu()
    named = torch.tensor([[3, 1, 0], [6, 0, 2]])
    for i in range(2):
        c, s, lo = fb.read_rows(kv[:, :, i], page, d, bool(i))
        assert torch.equal(got[:, :, i], (lo + s * c).to(F32).to(dtype)[named])


# ---- attention ----

def attention_bound(by_codes, by_values, want, dtype):
    """bfloat16: a rounding of each weight times its step (sum w (c - 8) + p (low + 8 step), where p stays float32: a relative 2^-8 of w moves that part alone), of the result, and, for portions, of keys and values (``cached``); float32 sums: scores of up to some 30 with
    errors of 2^-16, which are the relative errors of weights."""
    if dtype == F32:
        return 2.0 ** -14 * by_values + HALF[F32] * want.abs()
    return HALF[BF16] * (by_codes + want.abs()) + 2.0 ** -12 * by_values + 1e-30


def decode_case(lengths, nq, nkv, d, page, dtype, seed=0, lean=0.5):
    g = torch.Generator().manual_seed(seed)
    table, pages = fb.tables(lengths, page, g)
    kv = fb.random_cache(pages, nkv, page, d, g, lean)
    held = kv[..., page * d // 2:].contiguous().view(BF16)
    mask = torch.ones(pages, page, dtype=torch.bool)               # nobody's places stand for NaN
    for r, n in enumerate(lengths):
        for j in range(n):
            mask[table[r, j // page], j % page] = False
    held.view(pages, nkv, 2, page, -1)[mask[:, None, None].expand(-1, nkv, 2, -1)] = math.nan
    kv[..., page * d // 2:] = held.view(torch.uint8)
    q = torch.randn(len(lengths), nq * d, generator=g).to(dtype)
    return q.to(DEV), kv.to(DEV), table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)


HEADS = [(8, 2, 128, 64), (4, 4, 64, 16), (16, 1, 128, 16), (24, 2, 64, 128), (6, 1, 192, 32), (4, 1, 256, 64), (7, 1, 128, 64), (2, 1, 64, 4), (3, 1, 64, 1), (2, 2, 128, 3), (10, 2, 192, 2)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq,nkv,d,page", HEADS)
@pytest.mark.parametrize("lengths", [[1], [0], [63, 64, 65], [300, 0, 1, 16, 257], [2500]])
def test_decode(dtype, nq, nkv, d, page, lengths):
    q, kv, table, seq = decode_case(lengths, nq, nkv, d, page, dtype)
    want, by_codes, by_values = fb.attention(q, kv, table, [(1 if n else 0, n - 1 if n else 0) for n in lengths], nq, nkv, d, page, d ** -0.5)
    got = ops().attention_decode4(q, kv, table, seq, max(lengths), nq, nkv, d, page, d ** -0.5)
    within(got, want, attention_bound(by_codes, by_values, want, dtype))
    # a longer bound on the lengths, scratch and output of the caller's
    room = ops().decode4_scratch_floats(len(lengths), nq, nkv, d, table.shape[1] * page, page, dtype)
    out, scratch = torch.full_like(q, math.nan), torch.full((room + 1,), math.nan, device=DEV)
    again = ops().attention_decode4(q, kv, table, seq, table.shape[1] * page, nq, nkv, d, page, d ** -0.5, out, scratch)
    assert again.data_ptr() == out.data_ptr()
    within(out, want, attention_bound(by_codes, by_values, want, dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,nq,nkv,d,page", [(75, 16, 8, 128, 64), (75, 36, 4, 64, 16), (230, 6, 2, 128, 32), (60, 16, 8, 256, 64), (60, 8, 8, 192, 128)])
def test_decode_of_many_rows(dtype, rows, nq, nkv, d, page):
    """More pairs of a row and a kv head than three a multiprocessor, of ragged rows, some of them empty."""
    lengths = [(37 * r) % 211 if r % 9 else 0 for r in range(rows)]
    lengths[rows // 2] = 1500
    q, kv, table, seq = decode_case(lengths, nq, nkv, d, page, dtype)
    want, by_codes, by_values = fb.attention(q, kv, table, [(1 if n else 0, n - 1 if n else 0) for n in lengths], nq, nkv, d, page, d ** -0.5)
    got = ops().attention_decode4(q, kv, table, seq, max(lengths), nq, nkv, d, page, d ** -0.5)
    within(got, want, attention_bound(by_codes, by_values, want, dtype))
    assert torch.equal(got, ops().attention_decode4(q, kv, table, seq, max(lengths), nq, nkv, d, page, d ** -0.5))


@pytest.mark.parametrize("lengths", [[9000], [3000, 7, 5000], [100] * 70])
def test_decode_of_queries_of_any_size(lengths):
    """Queries times a power of two with the scale divided by it give the same bits, a head's own power among others'; a head of zeros has its values' mean."""
    nq, nkv, d, page = 16, 8, 128, 64
    q, kv, table, seq = decode_case(lengths, nq, nkv, d, page, BF16)
    run = lambda q, scale: ops().attention_decode4(q, kv, table, seq, max(lengths), nq, nkv, d, page, scale)
    want = run(q, d ** -0.5)
    for power in (-60, -9, 7, 60):
        assert torch.equal(run(q * 2.0 ** power, d ** -0.5 * 2.0 ** -power), want)
    heads = q.view(-1, nq, d).clone()
    heads[:, 3] *= 2.0 ** 30
    heads[:, 4] = 0
    got, kept = run(heads.view_as(q), d ** -0.5).view(-1, nq, d), [h for h in range(nq) if h // 2 not in (1, 2)]      # (heads of one kv head move their maxima together)
    assert torch.equal(got[:, kept], want.view(-1, nq, d)[:, kept]) and torch.isfinite(got).all()
    mean, by_codes, by_values = fb.attention(heads.view_as(q), kv, table, [(1, n - 1) for n in lengths], nq, nkv, d, page, d ** -0.5)
    bound = attention_bound(by_codes, by_values, mean, BF16)
    at = lambda x: x.view(-1, nq, d)[:, 4]
    within(got[:, 4], at(mean), at(bound))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_of_far_apart_scores(dtype):
    """Scores from -400 to 400: one place has all the weight, wherever it lies."""
    nq, nkv, d, page, n = 4, 1, 128, 64, 900
    for at in (0, 63, 64, 500, 899):
        q, kv, table, seq = decode_case([n], nq, nkv, d, page, dtype, seed=at)
        c, h = fb.hold(40.0 * q.float().cpu().view(nq, d)[0])
        fb.write_row(kv[table[0, at // page], 0, 0], at % page, page, d, False, c.to(DEV), h.to(DEV))
        want, by_codes, by_values = fb.attention(q, kv, table, [(1, n - 1)], nq, nkv, d, page, d ** -0.5)
        got = ops().attention_decode4(q, kv, table, seq, n, nq, nkv, d, page, d ** -0.5)
        # scores of 400 are off by up to 2^-24 of 400 in each of some 2^5 roundings: 2^-10 of a weight
        within(got, want, attention_bound(by_codes, by_values, want, dtype) + 2.0 ** -10 * by_values)


def test_decode_with_places_that_are_no_numbers():
    """A NaN key reaches its request's heads of that kv head, a NaN value the 64 features it stands for, and neither any other request."""
    nq, nkv, d, page = 8, 2, 128, 64
    for dtype in (BF16, F32):
        q, kv, table, seq = decode_case([200, 200, 200], nq, nkv, d, page, dtype)
        clean = ops().attention_decode4(q, kv, table, seq, 200, nq, nkv, d, page, d ** -0.5)
        nan = torch.full((2, 2), math.nan, dtype=BF16, device=DEV)
        zero = torch.zeros(d, dtype=torch.uint8, device=DEV)
        fb.write_row(kv[table[0, 1], 1, 0], 7, page, d, False, zero, nan)
        half = torch.tensor([[1.0, 0.0], [math.nan, math.nan]], dtype=BF16, device=DEV)
        fb.write_row(kv[table[2, 2], 0, 1], 9, page, d, True, zero, half)
        got = ops().attention_decode4(q, kv, table, seq, 200, nq, nkv, d, page, d ** -0.5).view(3, nkv, nq // nkv, d)
        bad = torch.zeros(3, nkv, nq // nkv, d, dtype=torch.bool, device=DEV)
        bad[0, 1] = True
        bad[2, 0, :, 64:] = True
        assert torch.equal(torch.isnan(got), bad)
        same = ~bad
        same[2, 0] = False                                  # (its other features see one value less)
        assert torch.equal(got[same], clean.view_as(got)[same])


PORTIONS = [([1], [0]), ([5], [0]), ([130], [0]), ([33, 1, 200], [0, 511, 70]), ([0, 64], [40, 64]), ([300], [700])]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq,nkv,d,page", [(8, 2, 128, 64), (4, 4, 64, 16), (24, 2, 64, 128), (4, 1, 256, 64), (3, 1, 192, 8)])
@pytest.mark.parametrize("new,cached", PORTIONS)
def test_portions(dtype, nq, nkv, d, page, new, cached):
    lengths = [p + n for p, n in zip(cached, new)]
    _, kv, table, _ = decode_case(lengths, nq, nkv, d, page, dtype, seed=2, lean=0.0)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(sum(new), nq * d, generator=g).to(dtype).to(DEV)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    pre = torch.tensor(cached, dtype=torch.int32, device=DEV)
    live = [i for i, n in enumerate(new) if n]
    want, by_codes, by_values = fb.attention(q, kv, table[live], [(new[i], cached[i]) for i in live], nq, nkv, d, page, d ** -0.5)
    got = ops().attention_prefill4(q, kv, table, cu, pre, cached, new, nq, nkv, d, page, d ** -0.5)
    bound = attention_bound(by_codes, by_values, want, dtype)
    if dtype == BF16:
        # keys rounded to bfloat16 move scores of |q| |k| d^-1/2 (up to some 4 |q_f k_f| sums) by 2^-8 of sum |q_f k_f| / sqrt(d), at most 2^-8 * 2 sqrt(d) here; weights and values are rounded too
        bound = bound + HALF[BF16] * (2 * 2 * d ** 0.5 + 2) * by_values
    within(got, want, bound)


def portions_case(new, cached, nq, nkv, d, page, seed=4):
    lengths = [p + n for p, n in zip(cached, new)]
    _, kv, table, _ = decode_case(lengths, nq, nkv, d, page, BF16, seed=seed, lean=0.0)
    q = torch.randn(sum(new), nq * d, generator=torch.Generator().manual_seed(seed)).to(BF16).to(DEV)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    pre = torch.tensor(cached, dtype=torch.int32, device=DEV)
    return q, kv, lambda q, kv, out=None, plan=None: ops().attention_prefill4(q, kv, table, cu, pre, cached, new, nq, nkv, d, page, d ** -0.5, out, plan), table


# both tensor-core kernels: many tokens and few, pages that the one takes and that only the other takes
WHO = [([700, 900, 600], [0, 130, 0], 8, 4, 128, 64), ([40, 1, 70], [3, 200, 0], 6, 2, 128, 16), ([30, 50, 9], [0, 20, 64], 4, 2, 192, 32), ([500, 700, 800], [10, 0, 100], 4, 4, 64, 64)]


@pytest.mark.parametrize("new,cached,nq,nkv,d,page", WHO)
def test_portions_keep_to_themselves(new, cached, nq, nkv, d, page):
    """Queries and keys of any size, and what is no number, change nothing in other requests' rows, in other tokens' rows above, or in other kv heads."""
    q, kv, run, table = portions_case(new, cached, nq, nkv, d, page)
    clean = run(q, kv)
    a, b = new[0], new[0] + new[1]
    for large in (3e38, 1e30, math.inf, math.nan):
        other = q.clone()
        other[a:b] = large                                     # a whole request
        assert torch.equal(run(other, kv)[:a], clean[:a]) and torch.equal(run(other, kv)[b:], clean[b:])
        other = q.clone()
        other[a - 1, d:2 * d] = large                          # one token's head
        got, kept = run(other, kv), torch.ones(a, nq, dtype=torch.bool, device=DEV)
        kept[a - 1, 1] = False
        assert torch.equal(got[:a].view(a, nq, d)[kept], clean[:a].view(a, nq, d)[kept]) and torch.equal(got[a:], clean[a:])
    # a key of the second request, in its kv head 1, whose lowest values are huge
    keys = kv.clone()
    held = torch.tensor([[1.0, 2.0 ** 100]] * (d // 64), dtype=BF16, device=DEV)
    fb.write_row(keys[table[1, 0], 1, 0], 0, page, d, False, torch.zeros(d, dtype=torch.uint8, device=DEV), held)
    got = run(q, keys)
    assert torch.equal(got[:a], clean[:a]) and torch.equal(got[b:], clean[b:])
    heads = slice(0, nq // nkv)
    assert torch.equal(got[a:b].view(-1, nq, d)[:, heads], clean[a:b].view(-1, nq, d)[:, heads])
    # rows behind the last portion
    room = torch.cat([q, torch.full((37, nq * d), 3e38, dtype=BF16, device=DEV)])
    out = torch.full_like(room, 7.0)
    run(room, kv, out)
    assert torch.equal(out[:len(q)], clean) and bool((out[len(q):] == 7.0).all())


@pytest.mark.parametrize("new,cached,nq,nkv,d,page", WHO)
def test_portions_of_queries_of_any_size(new, cached, nq, nkv, d, page):
    """A query head times a power of two, the keys divided by it, give the same bits; a head of zeros has the mean of the values it sees."""
    q, kv, run, table = portions_case(new, cached, nq, nkv, d, page)
    clean = run(q, kv)
    for power in (-40, 25):
        moved = kv.clone()
        held = moved[:, :, 0, page * d // 2:].contiguous().view(BF16)
        moved[:, :, 0, page * d // 2:] = (held * 2.0 ** -power).view(torch.uint8)
        assert torch.equal(run(q * 2.0 ** power, moved), clean)
    nothing = q.clone()
    nothing[3] = 0
    got = run(nothing, kv)
    want, by_codes, by_values = fb.attention(nothing, kv, table, list(zip(new, cached)), nq, nkv, d, page, d ** -0.5)
    # (weights and values are rounded: 2^-8 of the values' magnitudes each)
    within(got[3], want[3], HALF[BF16] * (2 * by_values[3] + want[3].abs()) + 2.0 ** -12 * by_values[3] + 1e-30)
    assert torch.equal(got[:3], clean[:3]) and torch.equal(got[4:], clean[4:])


def test_portions_refuse_a_plan_of_others():
    new, cached, nq, nkv, d, page = [40, 1, 70], [3, 200, 0], 6, 2, 128, 16
    q, kv, run, _ = portions_case(new, cached, nq, nkv, d, page)
    clean, plan = run(q, kv), lambda *a: ops().plan_prefill4(BF16, d, page, *a, q.device)
    assert torch.equal(run(q, kv, None, plan(cached, new)), clean)
    for other in (plan([0, 0, 0], [0, 0, 0]), plan(cached, [41, 1, 69]), plan([3, 216, 0], new), plan([19, 200, 0], new), ops().plan_prefill4(F32, d, page, cached, new, q.device)):
        if other.rows == plan(cached, new).rows and other.tile_req.numel() == plan(cached, new).tile_req.numel() and (other.pages, other.width) == plan(cached, new)[3:]:
            continue                                           # (lengths that are cut the same way)
        with pytest.raises(ops().KernelError, match="plan"):
            run(q, kv, None, other)


@pytest.mark.parametrize("page,planned", [(16, False), (16, True), (64, False), (64, True)])
def test_portions_in_a_graph(page, planned):
    """A captured call, its tiles a plan's or going with the launch; what is replayed follows the queries and the cache.  In float32 tiles are copied, so a call without a plan is refused."""
    new, cached, nq, nkv, d = [130, 1, 70], [3, 200, 0], 8, 2, 128
    q, kv, run, _ = portions_case(new, cached, nq, nkv, d, page)
    plan, out, stream = ops().plan_prefill4(BF16, d, page, cached, new, q.device) if planned else None, torch.zeros_like(q), torch.cuda.Stream()
    want, wide = [run(x, kv) for x in (q, q.flip(0).contiguous())], q.float()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            with pytest.raises(ops().KernelError, match="ahead of the capture"):
                run(wide, kv)
            run(q, kv, out, plan)
        graph.replay()
        stream.synchronize()
        assert torch.equal(out, want[0])
        q.copy_(q.flip(0).contiguous())
        graph.replay()
        stream.synchronize()
        assert torch.equal(out, want[1])


def test_portions_of_many_tiles():
    """More tiles than go with a launch: the same bits by a plan and without one, each request's as alone."""
    new, cached, nq, nkv, d, page = [1 + r % 3 for r in range(520)], [r % 40 for r in range(520)], 2, 1, 64, 16
    q, kv, run, table = portions_case(new, cached, nq, nkv, d, page)
    got = run(q, kv)
    assert torch.equal(run(q, kv, None, ops().plan_prefill4(BF16, d, page, cached, new, q.device)), got)
    want, by_codes, by_values = fb.attention(q, kv, table, list(zip(new, cached)), nq, nkv, d, page, d ** -0.5)
    # (test_portions says why: keys, weights and values are rounded)
    within(got, want, attention_bound(by_codes, by_values, want, BF16) + HALF[BF16] * (2 * 2 * d ** 0.5 + 2) * by_values)


# ---- streams, graphs, large offsets, together ----

def test_on_another_stream_and_in_a_graph():
    o = ops()
    nq, nkv, d, page = 8, 2, 128, 64
    q, kv, table, seq = decode_case([700, 33], nq, nkv, d, page, BF16)
    g = torch.Generator().manual_seed(3)
    codes, scales, z = fb.make_matrix(256, nq * d, 128, False, g, DEV)
    w = o.pack_weight4(codes, scales, z)

    def step():
        return o.linear4(o.attention_decode4(q, kv, table, seq, 700, nq, nkv, d, page, d ** -0.5), w)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    keep = q.clone()
    q.mul_(0.5)
    second = step()
    for graph in graphs:
        graph.replay()
    assert torch.equal(outs[0], second) and torch.equal(outs[1], second)
    q.copy_(keep)
    graphs[1].replay()
    graphs[0].replay()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_a_cache_beyond_32_bits():
    """Pages behind the first 2^32 bytes of a layer: written, read as numbers, attended to."""
    o = ops()
    nq, nkv, d, page = 8, 8, 128, 64
    per_page = nkv * 2 * page * (d // 2 + d // 16)
    pages = 2 ** 32 // per_page + 40
    kv = torch.zeros((pages, *o.cache4_shape(nkv, page, d)), dtype=torch.uint8, device=DEV)
    g = torch.Generator().manual_seed(1)
    c = write_case(BF16, nq, nkv, d, d, page, [100], [0], False, BF16, 4, kv=torch.zeros(4, nkv, 2, page * 72, dtype=torch.uint8))
    c["table"] = torch.tensor([[pages - 1, pages - 30]], dtype=torch.int32)
    small = dict(c, table=torch.tensor([[2, 1]], dtype=torch.int32))
    q_small, kv_small = run_write(small, nq, nkv, d, d, page, 1e-6)
    dev = {k: v.to(DEV) for k, v in c.items() if isinstance(v, torch.Tensor) and k != "kv"}
    q = o.qk_norm_rope_write4(dev["qkv"], None, None, 1e-6, dev["cos"], dev["sin"], dev["positions"], dev["req"], dev["table"], kv, nq, nkv, d, d, page)
    assert torch.equal(q.cpu(), q_small)
    assert torch.equal(kv[pages - 1].cpu(), kv_small[2]) and torch.equal(kv[pages - 30].cpu(), kv_small[1])
    seq = torch.tensor([100], dtype=torch.int32, device=DEV)
    far = o.attention_decode4(q[99:], kv, dev["table"], seq, 100, nq, nkv, d, page, d ** -0.5)
    near = o.attention_decode4(q[99:], kv_small.to(DEV), small["table"].to(DEV), seq, 100, nq, nkv, d, page, d ** -0.5)
    assert torch.equal(far, near)
    assert torch.equal(o.cache4_values(kv, dev["table"], nkv, d, page), o.cache4_values(kv_small.to(DEV), small["table"].to(DEV), nkv, d, page))
