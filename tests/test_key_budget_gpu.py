"""The kernels of a cache held to a budget of places, each against its definition in 64 bits: rotation by positions with several axes
into places of their own, attention that adds up what each key was given (one token a request; prompt portions), the choice of the
places that are kept and their move.  Pages are shuffled, what lies outside a request's places is NaN, and nothing outside them changes."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def ops():
    from lily_b200.csrc import ops as o
    return o


def close(got, want, dtype):
    """Sums of products in float32 (head sizes up to 256, scores up to about 30: an error of a score of some 1e-5, which is the
    relative error of a weight); bfloat16 results are rounded once, and so are the weights that meet bfloat16 values (2^-8 of values up to 4)."""
    tol = dict(atol=2e-2, rtol=1e-2) if dtype == BF16 else dict(atol=2e-5, rtol=1e-4)
    torch.testing.assert_close(got.double().cpu(), want.double().cpu(), equal_nan=True, **tol)


def pool(lengths, nkv, page, d, dtype, seed, lean=0.0):
    """(cache layer, weights, table): shuffled pages, NaN everywhere but in the requests' places."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    width, total = max(1, max(counts, default=1)), sum(counts) + 2
    order = torch.randperm(total, generator=g) + 1
    table = torch.zeros(len(lengths), width, dtype=torch.int32)
    kv = torch.full((total + 1, 2, nkv, page, d), math.nan)
    w = torch.full((total + 1, nkv, page), math.nan)
    at = 0
    for r, n in enumerate(lengths):
        table[r, :counts[r]] = order[at:at + counts[r]].int()
        at += counts[r]
        for j in range(0, n, page):
            p, m = int(table[r, j // page]), min(page, n - j)
            kv[p, :, :, :m] = torch.randn(2, nkv, m, d, generator=g)
            kv[p, 0, :, :m] += lean * torch.randn(nkv, m, 1, generator=g)
            w[p, :, :m] = torch.rand(nkv, m, generator=g)
    return kv.to(dtype).to(DEV), w.to(DEV), table.to(DEV)


def rows_of(x, table, r, n, page):
    """The first n places of request r of ``x`` [pages, ..., page, d] or [pages, nkv, page], as [nkv, n(, d)] in 64 bits."""
    p = table[r].long()[torch.arange(n, device=DEV) // page]
    off = torch.arange(n, device=DEV) % page
    return x[p, :, off].transpose(0, 1).double()


def put_rows(x, table, r, value, page):
    n = value.shape[1]
    p = table[r].long()[torch.arange(n, device=DEV) // page]
    x[p, :, torch.arange(n, device=DEV) % page] = value.transpose(0, 1).to(x.dtype)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0))


# ------------------------------------------------------------------------------ attention of one token a request

def decode_want(q, kv, w, table, lengths, nq, nkv, d, page, scale):
    out = torch.zeros(len(lengths), nq, d, dtype=torch.float64, device=DEV)
    w = w.double()
    group = nq // nkv
    for r, n in enumerate(lengths):
        if not n:
            continue
        k, v = rows_of(kv[:, 0], table, r, n, page), rows_of(kv[:, 1], table, r, n, page)
        p = torch.softmax(torch.einsum("ghd,gld->ghl", q[r].double().view(nkv, group, d), k) * scale, -1)
        out[r] = torch.einsum("ghl,gld->ghd", p, v).reshape(nq, d)
        old = rows_of(w, table, r, n, page)
        old[:, n - 1] = 0.0
        put_rows(w, table, r, old + p.sum(1), page)
    return out.reshape(len(lengths), nq * d), w


DECODE_SHAPES = [(16, 4, 128, 64), (32, 8, 128, 16), (8, 8, 64, 64), (14, 2, 64, 64), (40, 2, 128, 128), (6, 2, 48, 16), (20, 1, 96, 8), (3, 3, 256, 32), (5, 1, 7, 4)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nq,nkv,d,page", DECODE_SHAPES)
@pytest.mark.parametrize("lengths", [[1], [0, 1, 2, 63, 64, 65, 130], [700, 3, 0, 1999], [5000]])
def test_decode_weighed(dtype, nq, nkv, d, page, lengths):
    kv, w, table = pool(lengths, nkv, page, d, dtype, 3, lean=0.3)
    for r, n in enumerate(lengths):                               # the newest place's weight is whatever an earlier owner left
        if n:
            w[table[r, (n - 1) // page].long(), :, (n - 1) % page] = math.nan
    g = torch.Generator(device=DEV).manual_seed(5)
    q = (torch.randn(len(lengths), nq * d, device=DEV, generator=g) * 1.5).to(dtype)
    want, want_w = decode_want(q, kv, w, table, lengths, nq, nkv, d, page, d ** -0.5)
    seq = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got = ops().attention_decode_weighed(q, kv, w, table, seq, max(lengths), nq, nkv, d, page, d ** -0.5)
    close(got, want, dtype)
    close(w, want_w, F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nq,nkv,d,page,rows,longest", [(32, 8, 128, 64, 40, 1750), (16, 4, 64, 16, 70, 900), (16, 16, 128, 64, 3, 9000)])
def test_decode_weighed_of_many_or_long_rows(dtype, nq, nkv, d, page, rows, longest):
    lengths = [1 + (i * 7919) % longest for i in range(rows - 1)] + [longest]
    kv, w, table = pool(lengths, nkv, page, d, dtype, 11)
    q = torch.randn(rows, nq * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype)
    want, want_w = decode_want(q, kv, w, table, lengths, nq, nkv, d, page, d ** -0.5)
    scratch = torch.full((ops().decode_weighed_scratch_floats(rows, nq, nkv, d, longest + 13, page, dtype),), math.nan, device=DEV)
    out = torch.full_like(q, math.nan)
    seq = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    ops().attention_decode_weighed(q, kv, w, table, seq, min(longest + 13, table.shape[1] * page), nq, nkv, d, page, d ** -0.5, out=out, scratch=scratch)
    close(out, want, dtype)
    close(w, want_w, F32)


@pytest.mark.parametrize("dtype,d", [(F32, 128), (F32, 40), (BF16, 128), (BF16, 64), (BF16, 40)])
def test_decode_weighed_a_nan_key_reaches_its_row(dtype, d):
    lengths, page = [300, 300], 64
    kv, w, table = pool(lengths, 2, page, d, dtype, 2)
    kv[table[1, 3].long(), 0, 1, 7] = math.nan                    # request 1, kv head 1, place 199
    q = torch.randn(2, 4 * d, device=DEV).to(dtype)
    before = w.clone()
    out = ops().attention_decode_weighed(q, kv, w, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), 300, 4, 2, d, page, d ** -0.5).view(2, 2, 2, d)
    assert bool(torch.isnan(out[1, 1]).all()) and not bool(torch.isnan(out[0]).any()) and not bool(torch.isnan(out[1, 0]).any())
    assert bool(torch.isnan(rows_of(w, table, 1, 300, page)[1]).all())
    assert not bool(torch.isnan(rows_of(w, table, 1, 300, page)[0]).any()) and not bool(torch.isnan(rows_of(w, table, 0, 300, page)).any())
    assert same(w[0], before[0])


def test_decode_weighed_repeats_to_the_bit_and_on_another_stream():
    lengths = [4096, 77, 1300]
    kv, w, table = pool(lengths, 4, 64, 128, BF16, 8)
    q = torch.randn(3, 16 * 128, device=DEV).to(BF16)
    seq = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    a, b = w.clone(), w.clone()
    one = ops().attention_decode_weighed(q, kv, a, table, seq, 4096, 16, 4, 128, 64, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = ops().attention_decode_weighed(q, kv, b, table, seq, 4096, 16, 4, 128, 64, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(one, two) and same(a, b)


# ------------------------------------------------------------------------------ what a portion gives to the keys

def portion_want(q, kv, w, table, cached, new, nq, nkv, d, page, scale, observe):
    w, t0, group = w.double(), 0, nq // nkv
    for r, (p, n) in enumerate(zip(cached, new)):
        total, heard = p + n, min(n, observe or n)
        if not n:
            continue
        k = rows_of(kv[:, 0], table, r, total, page)
        x = q[t0 + n - heard:t0 + n].double().view(heard, nkv, group, d)
        s = torch.einsum("tghd,gld->ghtl", x, k) * scale
        own = torch.arange(total - heard, total, device=DEV)
        s = s.masked_fill(torch.arange(total, device=DEV)[None] > own[:, None], -math.inf)
        old = rows_of(w, table, r, total, page)
        old[:, p:] = 0.0
        put_rows(w, table, r, old + torch.softmax(s, -1).sum((1, 2)), page)
        t0 += n
    return w


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nq,nkv,d,page", [(16, 4, 128, 64), (8, 8, 64, 16), (14, 2, 64, 64), (6, 2, 128, 128), (32, 1, 128, 64), (6, 2, 48, 16), (3, 3, 96, 8), (5, 1, 7, 4)])
@pytest.mark.parametrize("cached,new,observe", [([0], [1], None), ([0, 5, 64], [65, 1, 63], None), ([129, 0], [200, 333], 32), ([700], [1], None), ([0], [600], None),
                                                ([1000, 0, 3], [130, 2, 300], 1), ([0, 200], [128, 129], 500)])
def test_key_weights(dtype, nq, nkv, d, page, cached, new, observe):
    lengths = [p + n for p, n in zip(cached, new)]
    kv, w, table = pool(lengths, nkv, page, d, dtype, 4, lean=0.3)
    for r, (p, n) in enumerate(zip(cached, new)):                 # what the portion's own places hold is nobody's
        for j in range(p, p + n):
            w[table[r, j // page].long(), :, j % page] = math.nan
    g = torch.Generator(device=DEV).manual_seed(6)
    q = (torch.randn(sum(new), nq * d, device=DEV, generator=g) * 1.5).to(dtype)
    want = portion_want(q, kv, w, table, cached, new, nq, nkv, d, page, d ** -0.5, observe)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    pre = torch.tensor(cached, dtype=torch.int32, device=DEV)
    ops().attention_key_weights(q, kv, w, table, cu, pre, cached, new, nq, nkv, d, page, d ** -0.5, observe=observe)
    close(w, want, F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cached,new,observe", [([0], [2048], None), ([6000], [700], 64), ([2000, 0, 31], [900, 1500, 40], None)])
def test_key_weights_of_long_portions(dtype, cached, new, observe):
    nq, nkv, d, page = 8, 2, 128, 64
    kv, w, table = pool([p + n for p, n in zip(cached, new)], nkv, page, d, dtype, 14, lean=0.5)
    q = torch.randn(sum(new), nq * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(6)).to(dtype)
    want = portion_want(q, kv, w, table, cached, new, nq, nkv, d, page, d ** -0.5, observe)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    pre = torch.tensor(cached, dtype=torch.int32, device=DEV)
    scratch = torch.full((ops().key_weights_scratch_floats(cached, new, nq, nkv, d, page, d ** -0.5, dtype, observe),), math.nan, device=DEV)
    again = w.clone()
    ops().attention_key_weights(q, kv, w, table, cu, pre, cached, new, nq, nkv, d, page, d ** -0.5, observe=observe, scratch=scratch)
    close(w, want, F32)
    ops().attention_key_weights(q, kv, again, table, cu, pre, cached, new, nq, nkv, d, page, d ** -0.5, observe=observe)
    assert same(w, again)                                         # to the bit: no sum depends on who comes first
    assert ops().key_weights_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_key_weights_of_large_scores(dtype):
    """Scores of several hundred, rising along the row: the running maximum moves in every tile, and most weights vanish."""
    nq, nkv, d, page, n = 4, 2, 128, 64, 500
    kv, w, table = pool([n], nkv, page, d, dtype, 1)
    for j in range(n):
        kv[table[0, j // page].long(), 0, :, j % page] = 0.02 * j
    q = torch.full((n, nq * d), 2.0, device=DEV).to(dtype)
    want = portion_want(q, kv, w, table, [0], [n], nq, nkv, d, page, d ** -0.5, None)
    cu, pre = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ops().attention_key_weights(q, kv, w, table, cu, pre, [0], [n], nq, nkv, d, page, d ** -0.5)
    # scores up to 226 are float32 numbers with an error of 1e-5 each: the weights' relative error is a few of those
    torch.testing.assert_close(w.double(), want, atol=1e-4, rtol=2e-4, equal_nan=True)


@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF16, 64), (BF16, 128), (BF16, 48)])
def test_key_weights_a_nan_key_reaches_its_rows(dtype, d):
    n, page = 300, 64
    kv, w, table = pool([n, n], 2, page, d, dtype, 2)
    kv[table[1, 4].long(), 0, 1, 3] = math.nan                    # request 1, kv head 1, place 259: rows 259 and up see it
    q = torch.randn(2 * n, 4 * d, device=DEV).to(dtype)
    cu, pre = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    ops().attention_key_weights(q, kv, w, table, cu, pre, [0, 0], [n, n], 4, 2, d, page, d ** -0.5)
    assert bool(torch.isnan(rows_of(w, table, 1, n, page)[1]).all())
    assert not bool(torch.isnan(rows_of(w, table, 1, n, page)[0]).any()) and not bool(torch.isnan(rows_of(w, table, 0, n, page)).any())


# ------------------------------------------------------------------------------ which places are kept

def select_want(w, table, lengths, keep, first, recent, page):
    kept = torch.full((w.shape[0], len(lengths), w.shape[2], keep), -1, dtype=torch.int32)
    for layer in range(w.shape[0]):
        for r, n in enumerate(lengths):
            for g, row in enumerate(rows_of(w[layer], table, r, n, page).tolist()):
                if n <= keep:
                    at = range(n)
                else:
                    middle = range(first, n - recent)
                    order = sorted(middle, key=lambda j: (-math.inf if math.isnan(row[j]) else -row[j], not math.isnan(row[j]), j))
                    at = sorted([*range(first), *order[:keep - first - recent], *range(n - recent, n)])
                kept[layer, r, g, :len(at)] = torch.tensor(list(at), dtype=torch.int32)
    return kept


@pytest.mark.parametrize("page", [4, 64])
@pytest.mark.parametrize("keep,first,recent", [(1, 0, 0), (7, 2, 3), (64, 4, 60), (300, 4, 32), (1024, 0, 1)])
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "strange"])
def test_select_keys(page, keep, first, recent, kind):
    lengths = [0, 1, keep - 1, keep, keep + 1, 2500, 513]
    _, w, table = pool(lengths, 3, page, 2, F32, 9)
    w = torch.stack([w, w.flip(1)])
    g = torch.Generator(device=DEV).manual_seed(1)
    if kind == "ties":
        w = torch.where(torch.isnan(w), w, torch.floor(w * 4) / 4)
    elif kind == "equal":
        w = torch.where(torch.isnan(w), w, 0.25)
    elif kind == "strange":
        odd = torch.tensor([math.inf, -math.inf, math.nan, -0.0, 0.0, -1.5, 1e-42, 3e38], device=DEV)
        w = torch.where(torch.rand(w.shape, device=DEV, generator=g) < 0.7, odd[torch.randint(0, 8, w.shape, device=DEV, generator=g)], w)
    got = ops().select_keys(w, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), max(lengths), keep, first, recent)
    assert torch.equal(got.cpu(), select_want(w, table, lengths, keep, first, recent, page))
    one = ops().select_keys(w[1].contiguous(), table, torch.tensor(lengths, dtype=torch.int32, device=DEV), max(lengths), keep, first, recent)
    assert torch.equal(one[0], got[1])


def test_select_keys_of_a_long_row():
    n, keep = 70001, 4097
    _, w, table = pool([n], 2, 64, 1, F32, 3)
    w = torch.where(torch.isnan(w), w, torch.floor(w * 5000) / 5000)[None].contiguous()
    got = ops().select_keys(w, table, torch.tensor([n], dtype=torch.int32, device=DEV), n, keep, 4, 100)
    assert torch.equal(got.cpu(), select_want(w, table, [n], keep, 4, 100, 64))


# ------------------------------------------------------------------------------ moving what is kept

def kept_lists(layers, lengths, nkv, keep, seed):
    g = torch.Generator().manual_seed(seed)
    kept = torch.full((layers, len(lengths), nkv, keep), -1, dtype=torch.int32)
    for layer in range(layers):
        for r, n in enumerate(lengths):
            for h in range(nkv):
                at = torch.randperm(n, generator=g)[:min(n, keep)].sort()[0]
                kept[layer, r, h, :len(at)] = at.int()
    return kept.to(DEV)


def move_want(x, table, to, kept, page):
    """``x`` [layers, pages, heads, page(, d)] after the move, from a copy of what it was."""
    out = x.clone()
    layers, requests, nkv, keep = kept.shape
    for layer in range(layers):
        for r in range(requests):
            for h in range(x.shape[2]):
                for i, j in enumerate(kept[layer, r, h % nkv].tolist()):
                    if j >= 0:
                        out[layer, to[r, i // page].long(), h, i % page] = x[layer, table[r, j // page].long(), h, j % page]
    return out


@pytest.mark.parametrize("fork", [False, True])
@pytest.mark.parametrize("dtype,d,page", [(BF16, 128, 64), (BF16, 64, 16), (F32, 128, 16), (BF16, 3, 4), (BF16, 6, 8), (F32, 5, 64), (BF16, 40, 16)])
@pytest.mark.parametrize("lengths,keep", [([150, 0, 1, 90], 90), ([300], 257), ([64, 65], 3), ([40], 64)])
def test_move_keys(fork, dtype, d, page, lengths, keep):
    layers, nkv = 2, 3
    both = lengths + [min(n, keep) for n in lengths]
    kv, w, table = zip(*[pool(both, nkv, page, d, dtype, 5) for _ in range(layers)])
    kv, w, table = torch.stack(kv), torch.stack(w), table[0]
    to = table[len(lengths):].contiguous()
    table = table[:len(lengths)].contiguous()
    kept = kept_lists(layers, lengths, nkv, keep, 1)
    target = to if fork else table
    want_kv = move_want(kv.view(layers, -1, 2 * nkv, page, d), table, target, kept, page).view_as(kv)
    want_w = move_want(w, table, target, kept, page)
    ops().move_keys(kv, w, table, kept, to_table=to if fork else None)
    assert same(kv, want_kv) and same(w, want_w)


def test_move_keys_in_place_over_many_tiles():
    """Long lists in place: what one tile of rows leaves must not meet what a later one reads, nor the other way round."""
    layers, nkv, page, d, n, keep = 1, 2, 64, 128, 9000, 6001
    kv, w, table = pool([n], nkv, page, d, BF16, 5)
    kept = kept_lists(layers, [n], nkv, keep, 2)
    kept[0, 0, 1] = torch.arange(keep, device=DEV) + 1            # every row one place down
    at = kept[0, 0].long()
    off, pages = at % page, table[0].long()[at // page]
    head = torch.arange(nkv, device=DEV)[:, None]
    want, want_w = kv[pages, :, head, off], w[pages, head, off]   # [nkv, keep, 2, d]
    ops().move_keys(kv, w, table, kept)
    i = torch.arange(keep, device=DEV)
    assert same(kv[table[0].long()[i // page], :, head, i % page], want) and same(w[table[0].long()[i // page], head, i % page], want_w)


def test_move_keys_without_weights_and_of_nothing():
    kv, w, table = pool([100], 2, 16, 8, BF16, 5)
    kept = kept_lists(1, [100], 2, 30, 1)
    want = move_want(kv.view(1, -1, 4, 16, 8), table, table, kept, 16)
    ops().move_keys(kv, None, table, kept)
    assert same(kv.view(1, -1, 4, 16, 8), want)
    ops().move_keys(kv, w, table, torch.full((1, 1, 2, 30), -1, dtype=torch.int32, device=DEV))
    assert same(kv.view(1, -1, 4, 16, 8), want)


# ------------------------------------------------------------------------------ rotation by several axes, into places

def rope_want(x, gain, cos, sin, positions, axis, rot, eps):
    x = x.double()
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    y = x.clone()
    for j in range(rot // 2):
        p = positions[axis[j]].long()
        c, s = cos[p, j].double()[:, None], sin[p, j].double()[:, None]
        y[..., j] = x[..., j] * c - x[..., j + rot // 2] * s
        y[..., j + rot // 2] = x[..., j + rot // 2] * c + x[..., j] * s
    return y


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("planes", [0, 1, 3, 9])
@pytest.mark.parametrize("gains", [None, F32, BF16])
@pytest.mark.parametrize("nq,nkv,d,rot,page,sections,in_turn", [(32, 8, 128, 128, 64, (16, 24, 24), False), (14, 2, 64, 64, 16, (8, 12, 12), True), (4, 4, 128, 64, 16, (11, 11, 10), True),
                                                              (2, 1, 96, 96, 8, (20, 28), False), (3, 1, 80, 32, 64, (16,), False), (2, 2, 10, 6, 4, (1, 0, 2), False), (1, 1, 7, 2, 4, (1,), True)])
def test_axes_rope_write(dtype, planes, gains, nq, nkv, d, rot, page, sections, in_turn):
    if dtype == F32 and gains == BF16:
        pytest.skip("float32 heads keep float32 gains")
    g = torch.Generator(device=DEV).manual_seed(21)
    new, cached = [1, 37, 5], [page - 1, 3, 2 * page]
    kv, _, table = pool([n + c for n, c in zip(new, cached)], nkv, page, d, dtype, 6)
    n, row = sum(new), (nq + 2 * nkv) * d
    qkv = torch.randn(planes, n, row, device=DEV, generator=g) if planes else torch.randn(n, row, device=DEV, generator=g).to(dtype)
    q_gain, k_gain = (None, None) if gains is None else ((1 + 0.3 * torch.randn(d, device=DEV, generator=g)).to(gains) for _ in range(2))
    angle = torch.outer(torch.arange(500.0, device=DEV), 1 / 100.0 ** (torch.arange(0, rot, 2, device=DEV) / rot))
    cos, sin = angle.cos(), angle.sin()
    positions = torch.randint(0, 500, (len(sections), n), device=DEV, generator=g, dtype=torch.int32)
    axis = ops().pair_axes(sections, DEV, in_turn)
    assert sorted(axis.tolist()) == [a for a, k in enumerate(sections) for _ in range(k)]
    places = torch.cat([c + torch.arange(m) for c, m in zip(cached, new)]).int().to(DEV)
    req = torch.repeat_interleave(torch.arange(3), torch.tensor(new)).int().to(DEV)
    x = (qkv.double().sum(0) if planes else qkv.double()).view(n, nq + 2 * nkv, d)
    want_kv = kv.double()
    pages, off = table.long()[req.long(), places.long() // page], places.long() % page
    want_kv[pages, 0, :, off] = rope_want(x[:, nq:nq + nkv], k_gain, cos, sin, positions, axis, rot, 1e-6)
    want_kv[pages, 1, :, off] = x[:, nq + nkv:]
    q = ops().axes_rope_write(qkv, q_gain, k_gain, 1e-6, cos, sin, positions, axis, places, req, table, kv, nq, nkv, d, rot, page)
    # one rounding of numbers up to about 8 (bfloat16: 2^-9 of them); float32: a few roundings of numbers up to 8
    tol = dict(atol=1e-3, rtol=2 ** -8) if dtype == BF16 else dict(atol=5e-6, rtol=5e-6)
    torch.testing.assert_close(q.double(), rope_want(x[:, :nq], q_gain, cos, sin, positions, axis, rot, 1e-6).reshape(n, -1), **tol)
    torch.testing.assert_close(kv.double(), want_kv, equal_nan=True, **tol)


def test_axes_rope_write_of_one_axis_is_the_written_rotation():
    """Where the place is the position and there is one axis: what ``qk_norm_rope_write`` leaves."""
    nq, nkv, d, page, n = 8, 2, 128, 64, 150
    g = torch.Generator(device=DEV).manual_seed(2)
    kv, _, table = pool([n], nkv, page, d, BF16, 6)
    other = kv.clone()
    qkv = torch.randn(n, (nq + 2 * nkv) * d, device=DEV, generator=g).to(BF16)
    gain = (1 + 0.3 * torch.randn(d, device=DEV, generator=g)).to(BF16)
    angle = torch.outer(torch.arange(200.0, device=DEV), 1 / 100.0 ** (torch.arange(0, d, 2, device=DEV) / d))
    at, req = torch.arange(n, device=DEV, dtype=torch.int32), torch.zeros(n, device=DEV, dtype=torch.int32)
    q = ops().axes_rope_write(qkv, gain, gain, 1e-6, angle.cos(), angle.sin(), at[None].contiguous(), ops().pair_axes((64,), DEV), at, req, table, kv, nq, nkv, d, d, page)
    p = ops().qk_norm_rope_write(qkv, gain, gain, 1e-6, angle.cos(), angle.sin(), at, req, table, other, nq, nkv, d, d, page)
    tol = dict(atol=1e-3, rtol=2 ** -7)                           # both round the same sums, whose last float32 bits may differ
    torch.testing.assert_close(q.float(), p.float(), **tol)
    torch.testing.assert_close(kv.float(), other.float(), equal_nan=True, **tol)


def test_axes_rope_write_outside_its_tables():
    nq, nkv, d, page = 2, 1, 128, 16
    kv, _, table = pool([20], nkv, page, d, BF16, 6)
    before = kv.clone()
    qkv = torch.randn(4, (nq + 2 * nkv) * d, device=DEV).to(BF16)
    angle = torch.rand(50, d // 2, device=DEV)
    positions = torch.tensor([[3, 50, 3, 3], [4, 4, -1, 4]], dtype=torch.int32, device=DEV)
    places = torch.tensor([1, 2, 3, 32], dtype=torch.int32, device=DEV)              # the last lies behind the table's two pages
    q = ops().axes_rope_write(qkv, None, None, 1e-6, angle.cos(), angle.sin(), positions, ops().pair_axes((32, 32), DEV), places,
                              torch.zeros(4, dtype=torch.int32, device=DEV), table, kv, nq, nkv, d, d, page).view(4, nq, 2, 2, 32)
    bad = torch.isnan(q.float())                                                   # [token, head, half, axis, pair]
    assert not bool(bad[0].any()) and not bool(bad[3].any())
    assert bool(bad[1, :, :, 0].all()) and not bool(bad[1, :, :, 1].any()) and bool(bad[2, :, :, 1].all()) and not bool(bad[2, :, :, 0].any())
    kv[table[0, 0].long(), :, :, 1:4] = before[table[0, 0].long(), :, :, 1:4]
    assert same(kv, before)


# ------------------------------------------------------------------------------ refusals

def test_what_is_refused():
    o = ops()
    nq, nkv, d, page = 4, 2, 64, 16
    kv, w, table = pool([40, 20], nkv, page, d, BF16, 1)
    q = torch.zeros(2, nq * d, device=DEV, dtype=BF16)
    seq = torch.tensor([40, 20], dtype=torch.int32, device=DEV)
    decode = lambda **k: o.attention_decode_weighed(**{**dict(q=q, kv_layer=kv, weights=w, block_table=table, seq_lens=seq, max_seq_len=40, nq=nq, nkv=nkv, d=d, page_size=page, scale=1.0), **k})
    for bad in (dict(q=q.float()), dict(q=q[:, :-d].contiguous()), dict(weights=w.double()), dict(weights=w[1:].contiguous()), dict(block_table=table[:1].contiguous()),
                dict(block_table=table.long()), dict(seq_lens=seq.long()), dict(max_seq_len=49), dict(nq=3), dict(q=q.cpu()), dict(q=q.t()), dict(scratch=torch.zeros(3, device=DEV)),
                dict(out=torch.zeros(2, nq * d, device=DEV)), dict(q=q.half(), kv_layer=kv.half())):
        with pytest.raises(o.KernelError):
            decode(**bad)
    wide = torch.zeros(3, 2, 1, 16, 264, device=DEV, dtype=BF16)
    with pytest.raises(o.KernelError, match="head size"):
        o.attention_decode_weighed(torch.zeros(1, 264, device=DEV, dtype=BF16), wide, torch.zeros(3, 1, 16, device=DEV), torch.ones(1, 1, device=DEV, dtype=torch.int32),
                                   torch.ones(1, device=DEV, dtype=torch.int32), 1, 1, 1, 264, 16, 1.0)
    x = torch.zeros(60, nq * d, device=DEV, dtype=BF16)
    cu, pre = torch.tensor([0, 40, 60], dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    portion = lambda **k: o.attention_key_weights(**{**dict(q=x, kv_layer=kv, weights=w, block_table=table, cu_seqlens=cu, prefix_lens=pre, h_prefix_lens=[0, 0], h_new_lens=[40, 20],
                                                            nq=nq, nkv=nkv, d=d, page_size=page, scale=1.0), **k})
    for bad in (dict(q=x.float()), dict(q=x[:50].contiguous()), dict(weights=w.bfloat16()), dict(cu_seqlens=cu[:2].contiguous()), dict(prefix_lens=pre.long()), dict(h_prefix_lens=[0]),
                dict(h_prefix_lens=[9, 0]), dict(observe=0), dict(observe=-1), dict(nkv=1), dict(scratch=torch.zeros(3, device=DEV)), dict(h_new_lens=[40, -1])):
        with pytest.raises(o.KernelError):
            portion(**bad)
    for bad in (dict(keep=0), dict(keep=4, first=3, recent=2), dict(first=-1), dict(max_length=49), dict(weights=w.double()), dict(lengths=seq.long()), dict(lengths=seq[:1])):
        with pytest.raises(o.KernelError):
            o.select_keys(**{**dict(weights=w, block_table=table, lengths=seq, max_length=40, keep=8, first=1, recent=1), **bad})
    kept = torch.zeros(1, 2, nkv, 4, dtype=torch.int32, device=DEV)
    for bad in (dict(kept=kept.long()), dict(kept=kept[:, :1].contiguous()), dict(kv=kv.half()), dict(weights=w.double()), dict(kept=kept[:, :, :1].contiguous()),
                dict(to_table=table[:1].contiguous()), dict(kv=kv[:, 0].contiguous())):
        with pytest.raises((o.KernelError, ValueError)):
            o.move_keys(**{**dict(kv=kv, weights=w, block_table=table, kept=kept), **bad})
    n = 3
    qkv = torch.zeros(n, (nq + 2 * nkv) * d, device=DEV, dtype=BF16)
    tab = torch.zeros(9, d // 2, device=DEV)
    i = torch.zeros(n, dtype=torch.int32, device=DEV)
    write = lambda **k: o.axes_rope_write(**{**dict(qkv=qkv, q_gain=None, k_gain=None, eps=1e-6, cos=tab, sin=tab, positions=i[None].contiguous(), pair_axis=o.pair_axes((d // 2,), DEV),
                                                    places=i, token_req=i, block_table=table, kv_layer=kv, nq=nq, nkv=nkv, d=d, rotary_dim=d, page_size=page), **k})
    gain = torch.ones(d, device=DEV)
    for bad in (dict(qkv=qkv[:, 8:].contiguous()), dict(cos=tab.bfloat16()), dict(cos=tab[:, 1:].contiguous()), dict(positions=i), dict(pair_axis=o.pair_axes((3,), DEV)), dict(places=i[:2].contiguous()),
                dict(places=i.long()), dict(q_gain=gain), dict(q_gain=gain, k_gain=gain.bfloat16()), dict(rotary_dim=d + 2), dict(qkv=qkv.half()), dict(nkv=1)):
        with pytest.raises(o.KernelError):
            write(**bad)
    with pytest.raises(o.KernelError):
        o.pair_axes((4, -1), DEV)
