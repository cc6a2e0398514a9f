"""The 4-bit cache: writing, reading back, attention, against 64 bits (tests/cache_reference.py)."""
import math

import pytest
import torch

from ptq_int8_lab_b200 import engine as E
from tests import cache_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ptq_int8_lab_b200.ops import Int8Ops
    with Int8Ops(0) as o:
        yield o


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def layout(g, lengths, page, spare=3, width=None):
    """(pages, table): every sequence's pages anywhere in the cache, arbitrary page names behind its last one."""
    need = [-(-max(0, n) // page) for n in lengths]
    pages = sum(need) + spare
    names = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.randint(0, pages, (len(lengths), width or max(1, max(need))), generator=g, device="cuda").to(torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = names[at:at + n]
        at += n
    return pages, table


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def begins(news):
    return ints([sum(news[:i]) for i in range(len(news) + 1)])


def random_cache(g, pages, kv, page, dim):
    from ptq_int8_lab_b200.ops import Cache4
    parts = []
    for off in (1.0, 0.3):
        codes = torch.randint(0, 256, (pages, kv, page, dim // 2), generator=g, device="cuda").to(torch.uint8)
        step = torch.rand((pages, kv, page, 1), generator=g, device="cuda") * 0.3 + 0.05
        least = -step * 7.5 + off * torch.randn((pages, kv, page, 1), generator=g, device="cuda")
        parts += [codes, torch.cat((step, least), -1).to(torch.bfloat16)]
    return Cache4(*parts)


TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("page,kv,lengths,news", [(16, 1, [1], [1]), (64, 8, [5, 700, 64], [3, 130, 0]), (32, 5, [33, 0, 31, 17], [33, 0, 1, 16]),
                                                  (256, 2, [1, 2, 3], None), (16, 3, [40, 16], [40, 2])])
def test_write_and_read(ops, dim, kind, page, kv, lengths, news):
    """Codes, steps and least values are the definition's, to the bit; what is read is their value; other rows are left alone."""
    g = generator(dim + page)
    counts = news or [1] * len(lengths)
    pages, table = layout(g, lengths, page)
    tokens = sum(counts)
    starts = begins(news) if news else None
    # both in one tensor, as a projection leaves them; one row constant, one tiny, one off zero
    both = torch.randn((tokens, 2 * kv + 1, dim), generator=g, device="cuda")
    both[0] = 0.375
    both[-1] *= 2.0 ** -120 if kind != "f16" else 2.0 ** -12
    both[tokens // 2] += 100.0
    both = both.to(TYPES[kind])
    k, v = both[:, :kv], both[:, kv:2 * kv]
    cache = random_cache(g, pages, kv, page, dim)
    before = [t.clone() for t in cache]
    ops.cache_write(cache, k, v, table, ints(lengths), starts)
    got = ops.cache_read(cache, table, ints(lengths), starts, tokens=tokens, dtype=torch.float32)
    at = 0
    for b, (n, length) in enumerate(zip(counts, lengths)):
        for i in range(n):
            pos = length - n + i
            name, place = int(table[b, pos // page]), pos % page
            for j, x in enumerate((k, v)):
                codes, step, least = R.quantized(x[at])
                c, s, l = R.rows_of(cache[2 * j][name, :, place], cache[2 * j + 1][name, :, place])
                assert torch.equal(c, codes) and torch.equal(s, step) and torch.equal(l, least)
                assert torch.equal(got[j][at].double(), (least + step * codes).float().double())
                before[2 * j][name, :, place] = cache[2 * j][name, :, place]
                before[2 * j + 1][name, :, place] = cache[2 * j + 1][name, :, place]
            at += 1
    assert all(torch.equal(a, b) for a, b in zip(before, cache))
    for name, t in TYPES.items():
        again = ops.cache_read(cache, table, ints(lengths), starts, tokens=tokens, dtype=t)
        assert all(torch.equal(a, b.to(t)) for a, b in zip(again, got))


@pytest.mark.parametrize("kind", list(TYPES))
def test_borders(ops, kind):
    """Values on and next to the border of two codes: the definition's 32-bit steps decide."""
    g = generator(3)
    t = TYPES[kind]
    x = (torch.randint(0, 31, (400, 2, 128), generator=g, device="cuda").float() * 0.5 * 0.3125 - 2.0)
    x[:, :, 0], x[:, :, 1] = -2.0, -2.0 + 15 * 0.3125
    x = torch.nextafter(x, x + torch.randint(-1, 2, x.shape, generator=g, device="cuda")) if kind == "f32" else x
    x = x.to(t)
    pages, table = layout(g, [400], 16)
    from ptq_int8_lab_b200.ops import new_cache
    cache = new_cache(pages, 2, 128, 16)
    ops.cache_write(cache, x, -x, table, ints([400]), begins([400]))
    k, v = ops.cache_read(cache, table, ints([400]), begins([400]), tokens=400, dtype=torch.float32)
    for got, want in ((k, x), (v, -x)):
        codes, step, least = R.quantized(want)
        assert torch.equal(got.double(), (least + step * codes).float().double())


def test_rows_that_are_not_finite(ops):
    """NaN, infinities and spreads beyond a float: NaN in the cache, for that row only."""
    g = generator(4)
    x = torch.randn((6, 2, 64), generator=g, device="cuda")
    x[1, 0, 5], x[2, 0, 0], x[3, 1, 63] = math.nan, math.inf, -math.inf
    x[4, 0, 0], x[4, 0, 1] = 3e38, -3e38
    from ptq_int8_lab_b200.ops import new_cache
    cache = new_cache(1, 2, 64, 16)
    ops.cache_write(cache, x, x, ints([[0]]), ints([6]), begins([6]))
    k, v = ops.cache_read(cache, ints([[0]]), ints([6]), begins([6]), tokens=6, dtype=torch.float32)
    bad = torch.zeros((6, 2), dtype=torch.bool, device="cuda")
    bad[1, 0] = bad[2, 0] = bad[3, 1] = bad[4, 0] = True
    for t in (k, v):
        assert torch.equal(torch.isnan(t).all(-1), bad) and torch.equal(torch.isnan(t).any(-1), bad)


def test_positions_without_a_page(ops):
    """Bad page names, positions behind the table and before 0, tokens of no sequence: skipped, zeros, left alone."""
    g = generator(5)
    from ptq_int8_lab_b200.ops import new_cache
    cache = new_cache(4, 1, 64, 16)
    table = ints([[2, -1], [4, 0], [1, 3]])
    lengths, starts = ints([20, 20, 40]), ints([2, 9, 29, 39])       # 7, 20 and 10 new tokens; 0, 1 and 39 .. 41 are of none
    k = torch.randn((42, 1, 64), generator=g, device="cuda")
    ops.cache_write(cache, k, k, table, lengths, starts)
    out = tuple(torch.full_like(k, 7.0) for _ in range(2))
    ops.cache_read(cache, table, lengths, starts, out=out)
    codes, step, least = R.quantized(k)
    want = (least + step * codes).float()
    want[:2] = want[39:] = 7.0
    want[2 + 3:9] = 0         # positions 13 .. 19 of sequence 0: 16 .. have page -1
    want[9:9 + 16] = 0        # sequence 1: page 4 of 4
    want[29 + 2:39] = 0       # positions 30 .. 39 of sequence 2: its table ends at 32
    assert all(torch.equal(t, want) for t in out)
    lengths = ints([3, 0, 1])  # fewer positions than new tokens: the first ones lie before 0
    ops.cache_write(cache, k, k, table, lengths, starts)
    ops.cache_read(cache, table, lengths, starts, out=out)
    want = (least + step * codes).float()
    want[:2] = want[39:] = 7.0
    want[2:2 + 4] = 0
    want[9:29] = 0
    want[29:38] = 0
    assert all(torch.equal(t, want) for t in out)


def check_attention(ops, g, kind, dim, kv, per, page, lengths, news, scale=None, cache=None, q=None, table=None, width=None):
    counts = news or [1] * len(lengths)
    pages, made = layout(g, lengths, page, width=width)
    table = made if table is None else table
    cache = cache or random_cache(g, pages, kv, page, dim)
    tokens = sum(counts)
    q = torch.randn((tokens, kv * per, dim), generator=g, device="cuda").to(TYPES[kind]) if q is None else q
    starts = begins(news) if news else None
    out = torch.full_like(q, 3.0)
    got = ops.cache_attention(q, cache, table, ints(lengths), starts, scale=scale, out=out)
    ops.check_device_error()
    assert got is out
    want, bound = R.attention(q, cache, table, ints(lengths), starts, dim ** -0.5 if scale is None else scale, torch.full_like(q, 3.0))
    far = (got.double() - want).abs()
    worst = float((far / bound).max())
    assert worst <= 1.0, (worst, float(far.max()))
    return got


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv,per", [(1, 1), (8, 4), (2, 8), (3, 6), (1, 16), (2, 12), (1, 32), (1, 71)])
def test_one_token(ops, kind, dim, kv, per):
    check_attention(ops, generator(per), kind, dim, kv, per, 64, [1, 63, 64, 65, 1000, 15, 16, 17], None)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv,per,page,lengths,news", [
    (2, 4, 16, [40, 300, 7, 1], [40, 2, 7, 1]), (1, 1, 32, [500], [500]), (3, 5, 64, [129, 0, 2000], [65, 0, 33]),
    (2, 2, 128, [1, 1, 128], [1, 1, 128]), (1, 16, 256, [777, 300], [3, 300]), (4, 3, 16, [2, 90, 33, 64, 65], [1, 9, 2, 0, 65])])
def test_pieces(ops, kind, dim, kv, per, page, lengths, news):
    check_attention(ops, generator(page + dim), kind, dim, kv, per, page, lengths, news)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_by_row_tile(ops, dim):
    """So many row tiles that none is cut."""
    rows = 64 if dim < 256 else 32
    n = 8 * 148 * 3 * rows // 32 + 5
    check_attention(ops, generator(dim), "bf16", dim, 8, 4, 64, [n // 4, n // 8, 3], [n // 4, n // 8, 3] if dim == 64 else [n // 4, n // 8, 3])


@pytest.mark.parametrize("length", [1, 2, 64, 4097, 40000])
def test_long_axis(ops, length):
    check_attention(ops, generator(length), "f16", 128, 1, 3, 64, [length], None)


def test_many_sequences(ops):
    g = generator(8)
    lengths = [int(v) for v in torch.randint(0, 300, (1024,), generator=g, device="cuda")]
    check_attention(ops, g, "bf16", 64, 2, 2, 16, lengths, None)
    news = [int(v) for v in torch.randint(0, 4, (1024,), generator=g, device="cuda")]
    check_attention(ops, g, "bf16", 64, 2, 2, 16, [max(a, b) for a, b in zip(lengths, news)], news)


def test_rows_that_see_nothing(ops):
    """Lengths of zero, fewer positions than new tokens, no page at all: zeros."""
    g = generator(9)
    got = check_attention(ops, g, "bf16", 128, 2, 4, 16, [0, 5, 0], None)
    assert not got[0].any() and got[1].any()
    got = check_attention(ops, g, "f16", 64, 2, 4, 16, [3, 40], [9, 5])
    assert not got[:6].any() and got[6:].any()
    cache = random_cache(g, 4, 2, 16, 64)
    got = check_attention(ops, g, "f16", 64, 2, 4, 16, [33, 50], [2, 3], cache=cache, table=ints([[-1, 4], [2, 7]]))
    assert not got[:2].any() and got[2:].any()


def test_width_of_the_table(ops):
    """A table much wider than the lengths, and lengths behind a table's end."""
    g = generator(10)
    check_attention(ops, g, "bf16", 128, 2, 2, 16, [30, 700], [3, 1], width=5000)
    cache = random_cache(g, 9, 2, 16, 64)
    table = torch.randint(0, 9, (2, 3), generator=g, device="cuda").to(torch.int32)
    check_attention(ops, g, "bf16", 64, 2, 2, 16, [60, 48], [20, 2], cache=cache, table=table)


def test_unseen_rows_may_hold_anything(ops):
    """NaN behind a sequence's end, in pages of others, and in positions after a query's own: no part in the output."""
    g = generator(11)
    lengths, news = [50, 90], [20, 1]
    pages, table = layout(g, lengths, 16)
    cache = random_cache(g, pages, 2, 16, 128)
    clean = [t.clone() for t in cache]
    used = torch.zeros((pages, 16), dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        for pos in range(n):
            used[table[b, pos // 16], pos % 16] = True
    for i in (1, 3):
        cache[i][~used.unsqueeze(1).expand(-1, 2, -1)] = math.nan
        clean[i][~used.unsqueeze(1).expand(-1, 2, -1)] = 0
    q = torch.randn((21, 8, 128), generator=g, device="cuda").to(torch.bfloat16)
    args = (table, ints(lengths), begins(news))
    assert torch.equal(ops.cache_attention(q, cache, *args), ops.cache_attention(q, clean, *args))
    # position 45 of sequence 0 becomes NaN: the tokens before it (30 .. 44) do not change, the others are NaN
    before = ops.cache_attention(q, cache, *args)
    name = int(table[0, 45 // 16])
    for i in (1, 3):
        saved = cache[i].clone()
        cache[i][name, 1, 45 % 16] = math.nan
        got = ops.cache_attention(q, cache, *args)
        assert torch.equal(got[:15], before[:15]) and torch.equal(got[:, :4], before[:, :4]) and torch.equal(got[20], before[20])
        assert torch.isnan(got[15:20, 4:]).all()
        cache[i].copy_(saved)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_sizes_far_apart(ops, kind):
    """Steps of differing magnitude, sharp and flat scores, queries of differing size, constant and zero rows."""
    g = generator(12)
    lengths = [600, 257]
    pages, table = layout(g, lengths, 64)
    cache = random_cache(g, pages, 2, 64, 128)
    for i, spread in ((1, 2.0), (3, 12.0)):
        cache[i].mul_((torch.rand(cache[i].shape[:3], generator=g, device="cuda")[..., None] * 2 * spread - spread).exp2().to(torch.bfloat16))
    cache[3][0] = 0      # values of zero
    cache[0][1] = 0      # keys that are constant
    q = torch.randn((2, 16, 128), generator=g, device="cuda") * torch.linspace(-12, 2, 16, device="cuda").exp2()[:, None]
    q[1, 3] = 0
    for scale in (None, 1.0, 0.0, -0.3):
        check_attention(ops, g, kind, 128, 2, 8, 64, lengths, None, scale=scale, cache=cache, q=q.to(TYPES[kind]), table=table)


def test_queries_that_are_not_finite(ops):
    g = generator(13)
    cache = random_cache(g, 3, 2, 64, 64)
    q = torch.randn((1, 8, 64), generator=g, device="cuda").to(torch.bfloat16)
    args = (ints([[0, 1, 2]]), ints([150]))
    good = ops.cache_attention(q, cache, *args)
    for value in (math.nan, math.inf, -math.inf):
        bad = q.clone()
        bad[0, 2, 7] = value
        got = ops.cache_attention(bad, cache, *args)
        assert torch.isnan(got[0, 2]).all()
        rest = [0, 1, 3, 4, 5, 6, 7]
        assert torch.equal(got[0, rest], good[0, rest])


def test_strides(ops):
    """Queries and outputs as parts of larger tensors at any element, caches as parts of one buffer, heads before pages."""
    g = generator(14)
    from ptq_int8_lab_b200.ops import Cache4
    lengths, news = [70, 33], [6, 3]
    pages, table = layout(g, lengths, 32)
    cache = random_cache(g, pages, 2, 32, 64)
    q = torch.randn((9, 6, 64), generator=g, device="cuda").to(torch.float16)
    args = (torch.cat((table, table), 1)[:, :table.shape[1]], ints(lengths), begins(news))
    want = ops.cache_attention(q, cache, *args)
    moved = Cache4(*(t.transpose(0, 1).contiguous().transpose(0, 1) for t in cache))
    big = torch.zeros((9, 7, 67), dtype=torch.float16, device="cuda")
    for off in (0, 1, 3):
        view = big[:, 1:, off:off + 64]
        view.copy_(q)
        assert torch.equal(ops.cache_attention(view, moved, *args), want)
        out = torch.zeros((9, 6, 69), dtype=torch.float16, device="cuda")
        ops.cache_attention(q, cache, *args, out=out[:, :, off:off + 64])
        assert torch.equal(out[:, :, off:off + 64], want) and not out[:, :, :off].any() and not out[:, :, off + 64:].any()
    k = torch.randn((9, 2, 64), generator=g, device="cuda")
    odd = torch.zeros((9, 3, 67), device="cuda")
    odd[:, :2, 3:] = k
    ops.cache_write(cache, k, k, *args)
    ops.cache_write(moved, odd[:, :2, 3:], odd[:, :2, 3:], *args)
    assert all(torch.equal(a, b) for a, b in zip(cache, moved))
    out = [torch.zeros((2, 9, 67), device="cuda")[:, :, 2:66].transpose(0, 1) for _ in range(2)]
    ops.cache_read(moved, *args, out=out)
    assert all(torch.equal(a, b) for a, b in zip(out, ops.cache_read(cache, *args, tokens=9, dtype=torch.float32)))


def test_the_same_twice(ops):
    """Nothing depends on which block comes first."""
    g = generator(15)
    lengths = [3000, 10, 700]
    pages, table = layout(g, lengths, 64)
    cache = random_cache(g, pages, 4, 64, 128)
    q = torch.randn((3, 16, 128), generator=g, device="cuda").to(torch.bfloat16)
    first = ops.cache_attention(q, cache, table, ints(lengths))
    for _ in range(20):
        assert torch.equal(ops.cache_attention(q, cache, table, ints(lengths)), first)
