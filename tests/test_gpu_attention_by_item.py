"""cache_attention with so many row tiles that each is a block's own (no shares, no parts, no workspace), on the kernel for few query rows."""
import pytest
import torch

from tests.test_gpu_cache import begins, check_attention, generator, ints, layout, ops, random_cache  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def by_item(ops, g, kind, dim, kv, per, page, lengths, news, **more):  # noqa: F811
    """Checks values, and that the call is one of these: only then is there no workspace."""
    pages, table = layout(g, lengths, page, width=more.get("width"))
    cache = random_cache(g, pages, kv, page, dim)
    q = torch.empty((sum(news), kv * per, dim), dtype={"f16": torch.float16, "bf16": torch.bfloat16}[kind], device="cuda")
    assert ops.cache_attention_workspace(q, cache, table, ints(lengths), begins(news)) == 0
    return check_attention(ops, g, kind, dim, kv, per, page, lengths, news, **more)


def test_one_prompt_of_256_dimensions(ops):  # noqa: F811
    """Tiles of 32 query rows, eight blocks an SM and more: the longest first."""
    n = -(-8 * sms() * 2 * 32 // 32) + 37
    by_item(ops, generator(1), "bf16", 256, 8, 4, 64, [n + 50], [n])


def test_prompts_of_256_dimensions(ops):  # noqa: F811
    """Sequences that end inside tiles, have nothing new, nothing at all, or see nothing with their first tokens."""
    n = -(-8 * sms() * 2 * 32 // 36)
    news = [n // 2, 0, 1, n // 4, 33, n // 4 + 8]
    by_item(ops, generator(2), "f16", 256, 4, 9, 16, [n // 2, 5, 400, n // 4 + 131, 20, n // 4 + 9], news)


@pytest.mark.parametrize("dim,per", [(64, 16), (64, 32), (128, 4), (128, 16), (256, 8), (256, 32)])
def test_single_tokens_with_starts(ops, dim, per):  # noqa: F811
    """A tile of 8, 16 or 32 rows a sequence and key head, two here and there and none elsewhere."""
    g = generator(dim + per)
    news = [(0 if i % 14 == 0 else 2) if i % 7 == 0 else 1 for i in range(1024)]
    lengths = [max(n, int(v)) for n, v in zip(news, torch.randint(0, 200, (1024,), generator=g, device="cuda"))]
    # `per` rows a sequence on average, or fewer: tiles of as many, or of 8; eight times as many of them as three blocks an SM
    assert sum(news) <= 1024
    kv = -(-8 * sms() * 3 // (sum(news) * per // max(8, per)))
    by_item(ops, g, "bf16", dim, kv, per, 16, lengths, news)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16)])
def test_short_pieces_of_many_sequences(ops, dim, page):  # noqa: F811
    """Tiles of 64 rows where a table has little room; the last tiles of sequences partly filled, some tokens before position 0."""
    g = generator(dim)
    most = 48
    tokens = -(-8 * sms() * 256 // 32) + 600   # heads 32: by item for tiles of 64 and of 256 rows
    each = -(-tokens // 1024)
    news = [each + (i % 5) - 2 for i in range(1024)]
    lengths = [min(most, max(0, n - 3 + int(v))) for n, v in zip(news, torch.randint(0, 40, (1024,), generator=g, device="cuda"))]
    assert sum(news) * 32 * most < (1 << 24 if dim == 128 else 1 << 25)   # fewer than tiles of 256 rows are taken for
    by_item(ops, g, "f16", dim, 2, 16, page, lengths, news)


def test_alone_and_beside_others(ops):  # noqa: F811
    """A sequence gives the same bits in a call of its own and beside others, again and again, captured and not."""
    g = generator(9)
    n = -(-8 * sms() * 2 * 32 // 32) + 5
    pages, table = layout(g, [n, 90], 64)
    cache = random_cache(g, pages, 8, 64, 256)
    q = torch.randn((n + 90, 32, 256), generator=g, device="cuda").to(torch.bfloat16)
    both = ops.cache_attention(q, cache, table, ints([n, 90]), begins([n, 90]))
    assert all(torch.equal(ops.cache_attention(q, cache, table, ints([n, 90]), begins([n, 90])), both) for _ in range(10))
    alone = ops.cache_attention(q[:n], cache, table[:1], ints([n]), begins([n]))
    assert torch.equal(alone, both[:n])
    graph = torch.cuda.CUDAGraph()
    out = torch.zeros_like(q)
    args = (q, cache, table, ints([n, 90]), begins([n, 90]))
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.cache_attention(*args, out=out)
    graph.replay()
    assert torch.equal(out, both)
    ops.check_device_error()
    del graph
