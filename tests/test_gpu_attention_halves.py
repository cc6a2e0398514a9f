"""cache_attention on tiles of 256 query rows: blocks whose tiles have one half of rows, then two, in all orders."""
import pytest
import torch

from tests.test_gpu_attention_tiles import ROOM, check
from tests.test_gpu_cache import begins, generator, ints, layout, ops, random_cache  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("per,news", [(4, [65] * 40), (4, [33, 65, 20, 96, 1, 64, 32, 97] * 6), (16, [17, 8, 16, 9, 24, 40] * 8)])
def test_halves_in_turn(ops, dim, per, news):  # noqa: F811
    """More row tiles than blocks; last tiles of one half beside full ones, of few and of many tiles of tokens."""
    g = generator(dim + per)
    extra = torch.randint(0, 700, (len(news),), generator=g, device="cuda").tolist()
    lengths = [n + (e if i % 3 else 0) for i, (n, e) in enumerate(zip(news, extra))]
    first = check(ops, g, "bf16", dim, 4, per, 64, lengths, news, width=ROOM // 64)
    assert bool(torch.isfinite(first).all())


@pytest.mark.parametrize("dim", [64, 128])
def test_halves_in_turn_repeat(ops, dim):  # noqa: F811
    g = generator(dim)
    news = [65, 20, 96, 33, 1, 200, 64] * 12
    lengths = [n + 37 * (i % 9) for i, n in enumerate(news)]
    pages, table = layout(g, lengths, 32, width=ROOM // 32)
    cache = random_cache(g, pages, 4, 32, dim)
    q = torch.randn((sum(news), 16, dim), generator=g, device="cuda").to(torch.float16)
    args = (q, cache, table, ints(lengths), begins(news))
    want = ops.cache_attention(*args)
    assert all(torch.equal(ops.cache_attention(*args), want) for _ in range(50))
    ops.check_device_error()
