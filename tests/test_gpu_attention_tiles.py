"""cache_attention on tiles of 256 query rows: calls that are taken there (many rows, a table with much room), against 64 bits."""
import math

import pytest
import torch

from ptq_int8_lab_b200 import engine as E
from tests import cache_reference as R
from tests.test_gpu_cache import TYPES, begins, generator, ints, layout, ops, random_cache  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu

def reference(q, cache, table, lengths, starts, scale, out):
    """(y, bound) of cache_reference, whose bound counts p step rounded to f16 as code p step 2^-11 a term.  A term enters these tiles
    as p step (code - 8), p not 1 even where one token is all that is seen: off by up to 8 p step 2^-11, whatever the code is.
    sum p step is what attention gives for codes of 1 and least values of 0.
    p step is f16 times a power of two that takes the largest step to 64 or more: what is below f16's normal numbers is off by half of
    2^-24, which is 2^-31 of that step, 8 times that for code - 8, for each token, over a sum of p that is 1 / 2 or more (references
    are whole numbers)."""
    steps = cache.v_scale[..., 0].double()
    finest = 2 * int(lengths.max()) * 8 * 2.0 ** -31 * float(steps[torch.isfinite(steps)].max())
    y, bound = R.attention(q, cache, table, lengths, starts, scale, out)
    ones = cache._replace(v=torch.full_like(cache.v, 0x11), v_scale=torch.cat((cache.v_scale[..., :1], torch.zeros_like(cache.v_scale[..., :1])), -1))
    return y, bound + 8 * 2.0 ** -11 * R.attention(q, ones, table, lengths, starts, scale, torch.zeros_like(out))[0] + finest


def check(ops, g, kind, dim, kv, per, page, lengths, news, scale=None, cache=None, q=None, table=None, width=None):  # noqa: F811
    pages, made = layout(g, lengths, page, width=width)
    table = made if table is None else table
    cache = cache or random_cache(g, pages, kv, page, dim)
    q = torch.randn((sum(news), kv * per, dim), generator=g, device="cuda").to(TYPES[kind]) if q is None else q
    args = (table, ints(lengths), begins(news))
    got = ops.cache_attention(q, cache, *args, scale=scale, out=torch.full_like(q, 3.0))
    ops.check_device_error()
    want, bound = reference(q, cache, *args, dim ** -0.5 if scale is None else scale, torch.full_like(q, 3.0))
    far = (got.double() - want).abs()
    assert bool((far <= bound).all()), (float((far / bound).max()), float(far.max()))
    return got


ROOM = 1 << 18   # tokens that the tables here have room for: enough for 128 rows and more


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv,per,page,lengths,news", [
    (2, 4, 64, [80], [80]),                       # nothing cached before, two halves of a tile
    (1, 1, 16, [1000], [130]),                    # pieces of a tile are pages
    (2, 8, 128, [3000, 77, 0, 400], [513, 70, 0, 9]),
    (3, 5, 32, [129, 2000], [129, 300]),          # rows that end inside a half
    (1, 71, 256, [777, 300], [300, 2]),           # heads that divide nothing
    (2, 32, 4096, [5000], [40]),
    (8, 4, 64, [128, 129, 255, 257], [128, 100, 255, 1]),
])
def test_pieces(ops, kind, dim, kv, per, page, lengths, news):  # noqa: F811
    check(ops, generator(page + dim), kind, dim, kv, per, page, lengths, news, width=ROOM // page)


@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_by_row_tile(ops, dim):  # noqa: F811
    """So many row tiles that none is cut."""
    n = 8 * 148 * 256 // 32 // 8 + 100
    check(ops, generator(dim), "bf16", dim, 8, 32, 64, [n + 50], [n], width=ROOM // 64)


@pytest.mark.parametrize("dim", [64, 128])
def test_one_token_of_many_heads(ops, dim):  # noqa: F811
    """No starts: a token's heads alone fill the tiles."""
    g = generator(8)
    lengths = [3000, 77, 0, 129]
    pages, table = layout(g, lengths, 64, width=ROOM // 64)
    cache = random_cache(g, pages, 1, 64, dim)
    q = torch.randn((4, 300, dim), generator=g, device="cuda").to(torch.bfloat16)
    got = ops.cache_attention(q, cache, table, ints(lengths), out=torch.full_like(q, 3.0))
    ops.check_device_error()
    want, bound = reference(q, cache, table, ints(lengths), None, dim ** -0.5, torch.full_like(q, 3.0))
    assert bool(((got.double() - want).abs() <= bound).all()) and not got[2].any()


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_see_nothing(ops, dim):  # noqa: F811
    g = generator(1)
    got = check(ops, g, "bf16", dim, 2, 4, 16, [60, 200], [100, 150], width=ROOM // 16)
    assert not got[:40].any() and got[40:].any()
    cache = random_cache(g, 20, 2, 16, dim)
    table = torch.full((2, ROOM // 16), -1, dtype=torch.int32, device="cuda")
    table[1, :8] = ints([3, -5, 20, 7, 1 << 30, 9, 0, 2])   # some of them no pages
    got = check(ops, g, "f16", dim, 2, 4, 16, [200, 130], [100, 120], cache=cache, table=table)
    assert not got[:100].any() and got[100:].any()


@pytest.mark.parametrize("dim", [64, 128])
def test_sizes_far_apart(ops, dim):  # noqa: F811
    g = generator(2)
    lengths, news = [700, 257], [90, 200]
    pages, table = layout(g, lengths, 64, width=ROOM // 64)
    cache = random_cache(g, pages, 2, 64, dim)
    for i, spread in ((1, 2.0), (3, 12.0)):
        cache[i].mul_((torch.rand(cache[i].shape[:3], generator=g, device="cuda")[..., None] * 2 * spread - spread).exp2().to(torch.bfloat16))
    cache[3][0] = 0
    cache[0][1] = 0
    q = torch.randn((290, 8, dim), generator=g, device="cuda") * torch.linspace(-12, 2, 8, device="cuda").exp2()[:, None]
    q[1, 3] = 0
    for scale in (None, 1.0, 0.0, -0.3):
        check(ops, g, "bf16", dim, 2, 4, 64, lengths, news, scale=scale, cache=cache, q=q.to(torch.bfloat16), table=table)


@pytest.mark.parametrize("dim", [64, 128])
def test_scores_that_grow(ops, dim):  # noqa: F811
    """The reference moves again and again, within a tile of tokens and between tiles."""
    g = generator(3)
    lengths, news = [900], [200]
    pages, table = layout(g, lengths, 64, width=ROOM // 64)
    cache = random_cache(g, pages, 1, 64, dim)
    for pos in range(900):   # constant keys of growing size: with queries of one sign their scores grow by some 0.3 a token
        cache[0][table[0, pos // 64].long(), 0, pos % 64] = 0
        cache[1][table[0, pos // 64].long(), 0, pos % 64, 1] = 0.02 * pos
    q = (torch.rand((200, 4, dim), generator=g, device="cuda") + 0.5).to(torch.bfloat16)
    check(ops, g, "bf16", dim, 1, 4, 64, lengths, news, cache=cache, q=q, table=table)
    check(ops, g, "bf16", dim, 1, 4, 64, lengths, news, cache=cache, q=-q, table=table)


@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_seen_and_what_is_not_finite(ops, dim):  # noqa: F811
    g = generator(4)
    lengths, news = [300], [100]
    pages, table = layout(g, lengths, 16, width=ROOM // 16)
    cache = random_cache(g, pages, 2, 16, dim)
    used = torch.zeros((pages, 16), dtype=torch.bool, device="cuda")
    for pos in range(300):
        used[table[0, pos // 16].long(), pos % 16] = True
    for i in (1, 3):
        cache[i][~used.unsqueeze(1).expand(-1, 2, -1)] = math.nan
    q = torch.randn((100, 8, dim), generator=g, device="cuda").to(torch.bfloat16)
    args = (table, ints(lengths), begins(news))
    want, bound = reference(q, cache, *args, dim ** -0.5, torch.zeros_like(q))
    at = 260   # the queries of positions 200 .. 259 do not see it
    name = int(table[0, at // 16])
    for i in (1, 3):
        for place in (0, 1):
            for value in (math.nan, math.inf, -math.inf, 2.0 ** 100):
                saved = cache[i].clone()
                cache[i][name, 1, at % 16, place] = value
                got = ops.cache_attention(q, cache, *args).double()
                cache[i].copy_(saved)
                assert bool(((got - want).abs() <= bound)[:60].all()) and bool(((got - want).abs() <= bound)[:, :4].all())
                assert not math.isnan(value) or torch.isnan(got[60:, 4:]).all()
    for value in (math.nan, math.inf, -math.inf):
        bad = q.clone()
        bad[7, 2, 5] = value
        got = ops.cache_attention(bad, cache, *args).double()
        assert torch.isnan(got[7, 2]).all()
        got[7, 2] = want[7, 2]
        assert bool(((got - want).abs() <= bound).all())
    ops.check_device_error()


def test_strides_and_rows_of_no_sequence(ops):  # noqa: F811
    g = generator(5)
    lengths, news = [500, 300], [120, 90]
    pages, table = layout(g, lengths, 32, width=ROOM // 32)
    cache = random_cache(g, pages, 2, 32, 128)
    q = torch.randn((220, 8, 128), generator=g, device="cuda").to(torch.float16)
    args = (table, ints(lengths), ints([3, 123, 213]))
    out = torch.full_like(q, 5.0)
    want = ops.cache_attention(q, cache, *args, out=out)
    assert bool((want[:3] == 5).all()) and bool((want[213:] == 5).all())
    big, moved = torch.zeros((220, 9, 131), dtype=torch.float16, device="cuda"), type(cache)(*(t.transpose(0, 1).contiguous().transpose(0, 1) for t in cache))
    for off in (0, 1, 3):
        view = big[:, 1:, off:off + 128]
        view.copy_(q)
        result = torch.full((220, 8, 133), 5.0, dtype=torch.float16, device="cuda")
        assert torch.equal(ops.cache_attention(view, moved, *args, out=result[:, :, off:off + 128]), want)
        assert bool((result[:, :, :off] == 5).all()) and bool((result[:, :, off + 128:] == 5).all())
    for _ in range(10):
        assert torch.equal(ops.cache_attention(q, cache, *args, out=out), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_attention(q, cache, *args, out=out)
    out.fill_(5.0)
    graph.replay()
    assert torch.equal(out, want)
    ops.check_device_error()
    del graph


def test_after_and_before_other_tensor_core_kernels(ops):  # noqa: F811
    """Kernels that hold TMEM follow one another without a pause."""
    from ptq_int8_lab_b200.ops import Int8Ops
    g = generator(6)
    pages, table = layout(g, [600], 64, width=ROOM // 64)
    cache = random_cache(g, pages, 2, 64, 64)
    q = torch.randn((300, 8, 64), generator=g, device="cuda").to(torch.bfloat16)
    x, xs = torch.randint(-127, 128, (300, 512), generator=g, device="cuda").to(torch.int8), torch.ones(300, device="cuda")
    w, ws = torch.randint(-127, 128, (1024, 512), generator=g, device="cuda").to(torch.int8), torch.ones(1024, device="cuda")
    want, product = ops.cache_attention(q, cache, table, ints([600]), begins([300])), ops.linear(x, xs, w, ws)
    lengths, starts = ints([600]), begins([300])
    got = [(ops.linear(x, xs, w, ws), ops.cache_attention(q, cache, table, lengths, starts)) for _ in range(30)]
    assert all(torch.equal(a, product) and torch.equal(b, want) for a, b in got)
    ops.check_device_error()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("per,lengths,news", [(4, [600], [200]), (64, [90], [80]), (16, [500, 40], [300, 40])])
def test_a_wait_runs_out(dim, per, lengths, news):
    from ptq_int8_lab_b200.ops import Int8Ops
    with Int8Ops(0) as ops:  # noqa: F811
        g = generator(7)
        pages, table = layout(g, lengths, 64, width=ROOM // 64)
        cache = random_cache(g, pages, 2, 64, dim)
        q = torch.randn((sum(news), 2 * per, dim), generator=g, device="cuda").to(torch.bfloat16)
        args = (q, cache, table, ints(lengths), begins(news))
        good = ops.cache_attention(*args)
        ops.check_device_error()
        ops.set_wait_test(10_000_000, True)
        ops.cache_attention(*args)
        with pytest.raises(E.Ptq8Error, match="ran out") as e:
            ops.check_device_error()
        assert e.value.status == 4
        ops.set_wait_test()
        assert torch.equal(ops.cache_attention(*args), good)
        ops.check_device_error()


@pytest.mark.parametrize("dim", [64, 128])
def test_two_streams_at_once(dim):
    """Tiles on one stream and tiles and products on another, each taking the tensor memory that the other leaves."""
    from ptq_int8_lab_b200.ops import Int8Ops
    with Int8Ops(0) as one, Int8Ops(0) as two:
        g = generator(9)
        pages, table = layout(g, [900], 64, width=ROOM // 64)
        cache = random_cache(g, pages, 2, 64, dim)
        q = torch.randn((400, 8, dim), generator=g, device="cuda").to(torch.bfloat16)
        x, xs = torch.randint(-127, 128, (300, 512), generator=g, device="cuda").to(torch.int8), torch.ones(300, device="cuda")
        w, ws = torch.randint(-127, 128, (1024, 512), generator=g, device="cuda").to(torch.int8), torch.ones(1024, device="cuda")
        args = (cache, table, ints([900]), begins([400]))
        want, product = one.cache_attention(q, *args), one.linear(x, xs, w, ws)
        need = one.cache_attention_workspace(q, *args)
        outs = [torch.zeros_like(q) for _ in range(2)]
        rooms = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
        y = torch.zeros_like(product)
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(40):
            one.cache_attention(q, *args, out=outs[0], workspace=rooms[0], stream=streams[0])
            two.linear(x, xs, w, ws, out=y, stream=streams[1])
            two.cache_attention(q, *args, out=outs[1], workspace=rooms[1], stream=streams[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want) and torch.equal(y, product)
        one.check_device_error(), two.check_device_error()
