"""Calls of the cache operators that are refused, and that a refused call leaves nothing behind; unusual sizes and strides that are not."""
import ctypes
import struct

import pytest
import torch

from ptq_int8_lab_b200 import engine as E
from tests import cache_reference as R
from tests.test_gpu_cache import begins, generator, ints, layout, random_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ptq_int8_lab_b200.ops import Int8Ops
    with Int8Ops(0) as o:
        yield o


def example(tokens=3, heads=4, kv=2, dim=64, page=16):
    g = generator(0)
    pages, table = layout(g, [20] * tokens, page)
    cache = random_cache(g, pages, kv, page, dim)
    return dict(q=torch.zeros((tokens, heads, dim), dtype=torch.float16, device="cuda"), k=torch.zeros((tokens, kv, dim), device="cuda"),
                cache=cache, table=table, lengths=ints([20] * tokens))


def test_refusals(ops):
    from ptq_int8_lab_b200.ops import Cache4
    e = example()
    c, table, lengths, q, k = e["cache"], e["table"], e["lengths"], e["q"], e["k"]

    def part(i, t):
        return Cache4(*(t if i == j else x for j, x in enumerate(c)))

    def other(pages, kv, page, dim):
        return random_cache(generator(1), pages, kv, page, dim)
    wide = torch.zeros((3, 2, 65), device="cuda")
    shared = [(dict(cache=part(0, c.k.to(torch.int8))), "cache.k"), (dict(cache=part(1, c.k_scale.float())), "cache.k_scale"), (dict(cache=part(2, c.v[:1])), "cache.v"),
              (dict(cache=part(3, c.v_scale.cpu())), "cpu"), (dict(cache=part(0, c.k[0])), "cache.k"), (dict(cache=part(0, c.k.transpose(2, 3).contiguous().transpose(2, 3))), "consecutive"),
              (dict(cache=part(0, torch.zeros(c.k.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(c.k.shape))), "16 bytes"),
              (dict(cache=part(0, c.k[:1].expand(c.k.shape))), "overlap"), (dict(cache=part(2, c.v[:, :1].expand(c.v.shape))), "overlap"),
              (dict(table=table.long()), "table"), (dict(table=table[0]), "table"), (dict(table=table.cpu()), "table"), (dict(table=table.t().contiguous().t()), "table"),
              (dict(table=table[:1].expand(table.shape)), "table_pitch"), (dict(lengths=lengths[:2]), "lengths"), (dict(lengths=lengths.long()), "lengths"), (dict(lengths=lengths.cpu()), "lengths"),
              (dict(starts=begins([1, 1])), "starts"), (dict(starts=begins([1, 1, 1]).long()), "starts"), (dict(table=table[:2], lengths=lengths[:2]), "without starts")]
    for change, text in shared + [(dict(k=k.double()), "dtype"), (dict(v=k.half()), "dtype"), (dict(k=k[:, :1]), "shape"), (dict(v=k[:2]), "shape"), (dict(k=k[0]), "shape"), (dict(k=k.cpu()), "cpu"),
                                  (dict(k=wide.transpose(1, 2)[:, :2].transpose(1, 2)), "shape"), (dict(v=torch.zeros((3, 2, 128), device="cuda")[:, :, ::2]), "columns"),
                                  (dict(cache=other(4, 2, 8, 64)), "page 8"), (dict(cache=other(4, 2, 48, 64)), "page 48"), (dict(cache=other(4, 2, 16, 96), k=torch.zeros((3, 2, 96), device="cuda"), v=torch.zeros((3, 2, 96), device="cuda")), "head_dim 96")]:
        args = dict(cache=c, k=k, v=k, table=table, lengths=lengths)
        args.update(change)
        with pytest.raises(E.Ptq8Error, match=text):
            ops.cache_write(**args)
        out = (args.pop("k").clone(memory_format=torch.preserve_format), args.pop("v"))
        if text != "columns":
            with pytest.raises(E.Ptq8Error, match=text):
                ops.cache_read(**args, out=out)
    for change, text in shared + [(dict(q=q.float()), "dtype"), (dict(q=q[:, :3]), "heads 3"), (dict(q=q[:, :, :32]), "shape"), (dict(q=q[0]), "shape"), (dict(q=q.cpu()), "cpu"),
                                  (dict(q=torch.zeros((3, 4, 128), dtype=torch.float16, device="cuda")[:, :, ::2], out=q), "columns"), (dict(out=q[:2]), "shape"), (dict(out=q.bfloat16()), "dtype"),
                                  (dict(out=q[:, :1].expand(q.shape)), "overlap"), (dict(out=q[:1].expand(q.shape)), "overlap"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
                                  (dict(workspace=torch.zeros(16, dtype=torch.uint8, device="cuda")), "workspace of 16"), (dict(workspace=torch.zeros(1 << 24, device="cuda")), "workspace"),
                                  (dict(workspace=torch.zeros(1 << 28, dtype=torch.uint8, device="cuda")[1:]), "aligned"), (dict(workspace=torch.zeros(1 << 20, dtype=torch.uint8)), "workspace"),
                                  (dict(stream=torch.cuda.current_stream()), "with stream")]:
        args = dict(q=q, cache=c, table=table, lengths=lengths)
        args.update(change)
        with pytest.raises(E.Ptq8Error, match=text):
            ops.cache_attention(**args)
    with pytest.raises(E.Ptq8Error, match="overlap"):
        ops.cache_read(c, table, lengths, out=(k, k[:, :1].expand(k.shape)))
    with pytest.raises(E.Ptq8Error, match="tokens"):
        ops.cache_read(c, table, lengths, begins([1, 1, 1]))
    with pytest.raises(E.Ptq8Error, match="dtype"):
        ops.cache_read(c, table, lengths, dtype=torch.int32)
    many = dict(table=table[:1].repeat(1025, 1), lengths=lengths[:1].repeat(1025))
    with pytest.raises(E.Ptq8Error, match="sequences 1025"):
        ops.cache_write(c, k[:1].repeat(1025, 1, 1), k[:1].repeat(1025, 1, 1), **many)
    ops.cache_attention(q, c, table, lengths)
    ops.check_device_error()


def test_refusals_of_the_entry_points(ops):
    """What only a C caller can pass: null pointers, negative numbers, types out of range."""
    from ptq_int8_lab_b200 import ops as module
    L, h = E.lib(), ops._h
    for call in (L.ptq8_cache_write, L.ptq8_cache_read, L.ptq8_cache_attention, L.ptq8_linear_w4):
        assert call(h, None, None) == 1
    assert L.ptq8_cache_attention_workspace(h, None) == -1
    e = example()
    fields = list(ops._cache(e["cache"], e["table"], e["lengths"], None, 3))
    k, q = e["k"], e["q"]
    rows = [k.data_ptr(), k.data_ptr(), *k.stride()[:2], *k.stride()[:2], 3, 0, 0]
    att = [q.data_ptr(), q.data_ptr(), *q.stride()[:2], *q.stride()[:2], 3, 0, 0, 0.125, 4, 1, 0]

    def refused(call, kind, values, at, value, text):
        values = list(values)
        values[at] = value
        buffer = ctypes.create_string_buffer(kind.pack(*values))
        assert call(h, buffer, None) == 1
        assert text in L.ptq8_ops_last_error(h), (text, L.ptq8_ops_last_error(h))
    n = len(fields)
    common = [(0, 0, b"null cache"), (3, 0, b"null cache"), (0, fields[0] + 8, b"16 bytes"), (4, 24, b"16 bytes"), (4, -fields[4], b"overlap"), (12, 0, b"null"), (12, fields[12] + 2, b"4 bytes"),
              (13, 0, b"table_pitch"), (14, 0, b"null"), (14, fields[14] + 1, b"4 bytes"), (15, 1, b"4 bytes"), (16, -1, b"pages"), (16, 1 << 31, b"pages"), (17, -1, b"table_width"),
              (17, 1 << 30, b"table_width"), (18, 0, b"page 0"), (18, 8192, b"page"), (18, -16, b"page"), (19, 0, b"kv_heads"), (19, -2, b"kv_heads"), (19, 1025, b"kv_heads"), (20, 0, b"head_dim"),
              (20, 512, b"head_dim"), (21, -1, b"sequences"), (21, 1025, b"sequences"), (21, 2, b"without starts")]
    for call, own in ((L.ptq8_cache_write, []), (L.ptq8_cache_read, [(n + 2, 1, b"overlap"), (n + 3, 1, b"overlap")])):
        for at, value, text in common + own + [(n, 0, b"null"), (n + 1, 0, b"null"), (n, rows[0] + 2, b"element type"), (n + 6, -1, b"tokens"), (n + 6, 1 << 40, b"tokens"), (n + 7, 3, b"type"), (n + 7, -1, b"type")]:
            refused(call, module._CACHE_ROWS, fields + rows, at, value, text)
    refused(L.ptq8_cache_write, module._CACHE_ROWS, fields + rows, n + 2, -1, b"negative")
    for at, value, text in common + [(n, 0, b"null"), (n + 1, 0, b"null"), (n, att[0] + 1, b"element type"), (n + 2, -1, b"negative"), (n + 4, 1, b"overlap"), (n + 6, -1, b"tokens"), (n + 9, float("inf"), b"scale"),
                                     (n + 10, 0, b"heads"), (n + 10, 4098, b"heads"), (n + 11, 0, b"type"), (n + 11, 3, b"type"), (n, att[0], b"workspace")]:
        refused(L.ptq8_cache_attention, module._ATTENTION, fields + att, at, value, text)
    w4 = struct.Struct(module._W4.format)
    w, s, x = torch.zeros((8, 32), dtype=torch.uint8, device="cuda"), torch.ones((8, 1), device="cuda"), torch.zeros((2, 64), device="cuda")
    good = [x.data_ptr(), 64, w.data_ptr(), 32, s.data_ptr(), 1, 0, x.data_ptr(), 64, 2, 64, 8, 64, 0, 0, 0, 0, 0]
    for at, value, text in ((0, 0, b"null"), (2, 0, b"null"), (4, 0, b"null"), (7, 0, b"null"), (0, good[0] + 1, b"element type"), (6, 1, b"element type"), (1, 63, b"ldx"), (3, 31, b"ldw"), (5, 0, b"lds"),
                            (8, 7, b"ldy"), (9, -1, b"rows"), (10, 0, b"in_features"), (10, 1 << 25, b"in_features"), (11, 0, b"out_features"), (11, -1, b"out_features"), (12, 0, b"group"), (12, -32, b"group"),
                            (13, 2, b"epilogue"), (14, 3, b"x_type"), (15, -1, b"scale_type"), (16, 7, b"y_type")):
        refused(L.ptq8_linear_w4, w4, good, at, value, text)
    ops.check_device_error()


def test_nothing_to_do(ops):
    """No tokens, no sequences, no pages, a table without columns."""
    from ptq_int8_lab_b200.ops import new_cache
    for pages in (0, 2):
        cache = new_cache(pages, 2, 64, 16)
        none = ints([]).view(0, 3)
        k, q = torch.zeros((0, 2, 64), device="cuda"), torch.zeros((0, 4, 64), dtype=torch.float16, device="cuda")
        ops.cache_write(cache, k, k, none, ints([]))
        ops.cache_read(cache, none, ints([]))
        assert ops.cache_attention(q, cache, none, ints([])).shape == q.shape
        three, out = torch.ones((3, 2, 64), device="cuda"), torch.ones((3, 4, 64), dtype=torch.float16, device="cuda")
        for table in (ints([[0, 1], [5, -1], [-7, 2]]) - (3 if pages else 0), ints([]).view(3, 0)):   # no page of the cache among them
            n = ints([2, 3, 1])
            ops.cache_write(cache, three, three, table, n)
            assert not any(t.any() for t in ops.cache_read(cache, table, n))
            assert not ops.cache_attention(out, cache, table, n).any()
        assert not any(t.any() for t in cache)
        # tokens of no sequence
        left = ops.cache_attention(out, cache, none, ints([]), ints([0]), out=out.clone())
        assert torch.equal(left, out)
    ops.check_device_error()


def test_starts_that_are_wrong(ops):
    """Values outside are clamped; where they decrease, no access leaves the tensors."""
    g = generator(2)
    pages, table = layout(g, [40] * 4, 16)
    cache = random_cache(g, pages, 2, 16, 64)
    q = torch.randn((7, 8, 64), generator=g, device="cuda").to(torch.float16)
    k = torch.randn((7, 2, 64), generator=g, device="cuda")
    clamped = ops.cache_attention(q, cache, table, ints([40] * 4), ints([-5, 3, 3, 5, 900]))
    assert torch.equal(clamped, ops.cache_attention(q, cache, table, ints([40] * 4), ints([0, 3, 3, 5, 7])))
    around = torch.full((9, 8, 64), 7.0, dtype=torch.float16, device="cuda")
    for starts in ([7, 0, 7, 0, 7], [0, 7, 0, 7, 0], [-2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 0], [5, 4, 3, 2, 1]):
        ops.cache_attention(q, cache, table, ints([40] * 4), ints(starts), out=around[1:8])
        assert bool((around[0] == 7).all()) and bool((around[8] == 7).all())
        ops.cache_write(cache, k, k, table, ints([40] * 4), ints(starts))
        ops.cache_read(cache, table, ints([40] * 4), ints(starts), tokens=7)
    ops.check_device_error()


def test_lengths_past_everything(ops):
    """Lengths that the table has no room for, and below zero."""
    g = generator(3)
    pages, table = layout(g, [64] * 3, 16)
    cache = random_cache(g, pages, 1, 16, 128)
    q = torch.randn((3, 8, 128), generator=g, device="cuda").to(torch.bfloat16)
    y = ops.cache_attention(q, cache, table, ints([2 ** 31 - 1, 64, -2 ** 31]))
    want = ops.cache_attention(q, cache, table, ints([64, 64, 64]))
    assert torch.equal(y[:2], want[:2]) and not y[2].any()
    k = torch.ones((3, 1, 128), device="cuda")
    before = [t.clone() for t in cache]
    ops.cache_write(cache, k, k, table, ints([2 ** 31 - 1, 65, -2 ** 31]))
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    ops.check_device_error()


def test_offsets_past_32_bits(ops):
    """Pages, tokens and outputs more than 2^32 bytes (and 2^31 elements) apart."""
    from ptq_int8_lab_b200.ops import Cache4
    g = generator(4)
    far, page, kv, dim = (1 << 32) + 512, 16, 2, 64
    small = random_cache(g, 2, kv, page, dim)
    buffer = torch.empty(far + (1 << 20), dtype=torch.uint8, device="cuda")
    at, parts = 0, []
    for t in small:
        size = t.element_size()
        view = buffer.view(t.dtype).as_strided(t.shape, (far // size, *t.stride()[1:]), at // size)
        view.copy_(t)
        parts.append(view)
        at += t[0].numel() * size
    cache = Cache4(*parts)
    table, lengths = ints([[1, 0]]), ints([27])
    q = torch.randn((2, 4, dim), generator=g, device="cuda").to(torch.bfloat16)
    starts = begins([2])
    want = ops.cache_attention(q, small, table, lengths, starts)
    assert torch.equal(ops.cache_attention(q, cache, table, lengths, starts), want)
    # the token stride: 2^31 + 64 elements of bf16 past the pages' parts
    wide = torch.empty((1 << 31) + (1 << 16), dtype=torch.bfloat16, device="cuda")
    qs, out = (wide.as_strided((2, 4, dim), ((1 << 31) + 64, dim, 1), first) for first in (0, 1024))
    qs.copy_(q)
    ops.cache_attention(qs, cache, table, lengths, starts, out=out)
    assert torch.equal(out, want)
    k, v = (wide.as_strided((2, kv, dim), ((1 << 31) + 64, dim, 1), first) for first in (2048, 4096))
    k.copy_(torch.randn((2, kv, dim), generator=g, device="cuda")), v.copy_(torch.randn((2, kv, dim), generator=g, device="cuda"))
    ops.cache_write(small, k.contiguous(), v.contiguous(), table, lengths, starts)
    ops.cache_write(cache, k, v, table, lengths, starts)
    assert all(torch.equal(a, b) for a, b in zip(cache, small))
    want = ops.cache_read(small, table, lengths, starts, tokens=2)
    ops.cache_read(cache, table, lengths, starts, out=(k, v))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    ops.check_device_error()


def test_many_tokens_of_linear_w4(ops):
    """Far more tokens than a pass takes, odd in number: each is what it is in a call of a few."""
    g = generator(5)
    w, s = torch.randint(0, 256, (72, 128), generator=g, device="cuda").to(torch.uint8), torch.rand((72, 4), generator=g, device="cuda")
    x = torch.randn((2501, 256), generator=g, device="cuda").to(torch.bfloat16)
    y = ops.linear_w4(x, w, s, 64)
    codes = torch.stack((w & 15, w >> 4), -1).flatten(1).double()
    full = torch.where(codes > 7, codes - 16, codes) * s.double().repeat_interleave(64, 1)
    want = x.double() @ full.t()
    # the output's rounding, and f32 sums of at most 256 terms cut or rounded at 2^-23 of the terms' sum each
    allowed = 2.0 ** -8 * want.abs() + 256 * 2.0 ** -23 * (x.double().abs() @ full.abs().t())
    assert bool(((y.double() - want).abs() <= allowed).all())


def test_reference_agrees_with_the_definition():
    """The 64-bit forms here, against a loop over single numbers."""
    x = torch.tensor([[0.0, 1.0, -3.0, 2.5] + [0.25] * 60])
    codes, step, least = R.quantized(x)
    assert float(least) == -3.0 and float(step) == 0.3671875   # 5.5 / 15 = 0.36667, up to bf16: 0.3671875
    assert [int(c) for c in codes[0, :4]] == [8, 11, 0, 15]
