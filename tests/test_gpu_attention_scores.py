"""cache_attention where scores are far larger than usual, or far apart: few query rows and tiles of many, against 64 bits."""
import math

import pytest
import torch

from tests import cache_reference as R
from tests.test_gpu_cache import TYPES, begins, generator, ints, layout, ops, random_cache  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu

ROOM = 1 << 18   # tokens that a table has room for: tiles of 256 rows where a sequence has more than 64
CASES = [(64, 2, 0), (128, 2, 0), (256, 2, 0), (128, 40, 0), (64, 100, ROOM), (128, 100, ROOM), (256, 100, 0)]   # dim, new tokens, room


def expected(q, cache, table, length, news, scale):
    """(y, bound) like q in 64 bits for one sequence of whole pages.  Scores are off by delta: sums of dim products and a few more
    roundings of 2^-23 of their terms' magnitudes, counted where a token's p is more than 2^-60 (elsewhere p stays nothing), and
    not where all such tokens' keys are the same, whose scores are off alike.  A term enters as p step (code - 8), p step rounded to f16 (2^-11, and 2^-31 of the largest step that is seen as its finest), beside
    p (least + 8 step) in f32."""
    page, kv, dim = cache[0].shape[2], cache[0].shape[1], q.shape[2]
    per = q.shape[1] // kv
    (kc, ks, kl), (vc, vs, vl), _ = R.gathered(cache, table[0], length, page)
    y, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    seen = torch.arange(length, device="cuda")[None] <= torch.arange(length - news, length, device="cuda")[:, None]
    for h in range(kv):
        x = q[:, h * per:(h + 1) * per].double()
        z = torch.einsum("npd,jd->npj", x, kc[:, h] * ks[:, h] + kl[:, h]) * scale
        size = torch.einsum("npd,jd->npj", x.abs(), kc[:, h] * ks[:, h].abs() + kl[:, h].abs()) * abs(scale)
        z = z.masked_fill(~seen[:, None], -math.inf)
        z = z - z.amax(-1, keepdim=True)
        p = torch.exp(z)
        delta = ((dim + 16) * 2.0 ** -23 * size).masked_fill(p < 2.0 ** -60, 0).amax(-1, keepdim=True)
        delta = torch.where(((p >= 2.0 ** -60) & (z < 0)).any(-1, keepdim=True), delta, 0.0)
        p = p / p.sum(-1, keepdim=True)
        v = vc[:, h] * vs[:, h] + vl[:, h]
        y[:, h * per:(h + 1) * per] = p @ v
        steps = (p @ vs[:, h]) * 8
        adds = length / 16 + 64
        bound[:, h * per:(h + 1) * per] = (torch.finfo(q.dtype).eps / 2 * 1.01 * (p @ v).abs() + 2.0 ** -11 * steps + 2 * length * 8 * 2.0 ** -31 * vs.max()
                                           + (adds * 2.0 ** -22 + 2.5 * delta) * (p @ (v.abs() + 8 * vs[:, h])))
    return y, bound + 2.0 ** -24


def constant_keys(cache, table, values):
    """The keys of position i become values[i] in every dimension (values: f32 that bf16 holds); codes of zero."""
    page = cache[0].shape[2]
    at = torch.arange(values.numel(), device="cuda")
    name = table[0].long()[at // page]
    cache[0][name, :, at % page] = 0
    cache[1][name, :, at % page, 0] = 0.0
    cache[1][name, :, at % page, 1] = values.to(torch.bfloat16)[:, None]


def run(ops, g, dim, news, room, length, keys, q_value, kind="bf16", scale=None):  # noqa: F811
    page = 64
    pages, table = layout(g, [length], page, width=max(room // page, -(-length // page)))
    cache = random_cache(g, pages, 2, page, dim)
    constant_keys(cache, table, keys)
    q = torch.full((news, 8, dim), q_value, device="cuda").to(TYPES[kind])
    got = ops.cache_attention(q, cache, table, ints([length]), begins([news]), scale=scale)
    ops.check_device_error()
    want, bound = expected(q, cache, table, length, news, dim ** -0.5 if scale is None else scale)
    far = (got.double() - want).abs()
    assert bool((far <= bound).all()), (float((far / bound).max()), float(far.max()))


@pytest.mark.parametrize("dim,news,room", CASES)
@pytest.mark.parametrize("top", [1.0, 2.0 ** 100, 2.0 ** 103])
def test_all_scores_far_below_zero(ops, dim, news, room, top):  # noqa: F811
    """However low they are, the largest ones have the weight (ties: the same)."""
    g = generator(dim + news)
    length = 500
    keys = -top * (torch.randint(2, 9, (length,), generator=g, device="cuda").float())
    keys[5], keys[200], keys[390] = -top, -top, -top
    run(ops, g, dim, news, room, length, keys, 1.0)


@pytest.mark.parametrize("dim,news,room", CASES)
@pytest.mark.parametrize("scale", [None, 0.3, -0.7])
@pytest.mark.parametrize("top", [2.0 ** 16, 2.0 ** 24, 2.0 ** 30, 2.0 ** 60, 2.0 ** 100])
def test_large_scores(ops, dim, news, room, top, scale):  # noqa: F811
    """Scores of any size: the largest ones share the weight, wherever they lie."""
    g = generator(dim + news)
    length = 500
    keys = top * torch.randint(-8, 9, (length,), generator=g, device="cuda").float()
    run(ops, g, dim, news, room, length, keys, 1.0, scale=scale)
    keys = top * (1 + torch.arange(length, device="cuda") // 90 / 128)   # growing, each of them a hundred times
    run(ops, g, dim, news, room, length, keys, 1.0, scale=scale)


@pytest.mark.parametrize("dim,news,room", CASES)
@pytest.mark.parametrize("low", [2.0 ** 10, 2.0 ** 17, 2.0 ** 20, 2.0 ** 30, 2.0 ** 80])
@pytest.mark.parametrize("first", [16, 40, 128, 300])
def test_ordinary_scores_after_far_lower_ones(ops, dim, news, room, low, first):  # noqa: F811
    g = generator(first)
    length = 450
    keys = torch.randn(length, generator=g, device="cuda").to(torch.bfloat16).float() * 0.25
    keys[:first] = -low * (1 + torch.arange(first, device="cuda") % 3)
    run(ops, g, dim, news, room, length, keys, 1.0)
    keys = keys.flip(0)
    run(ops, g, dim, news, room, length, keys, 1.0)


@pytest.mark.parametrize("dim,news,room", CASES)
@pytest.mark.parametrize("exponent", [-120, -110, -60, 60, 115, 117, 120, 126])
def test_queries_of_any_size(ops, dim, news, room, exponent):  # noqa: F811
    """Queries over bf16's range, keys so that the scores are ordinary ones: as accurate as any."""
    g = generator(dim + news)
    length, page = 500, 64
    pages, table = layout(g, [length], page, width=max(room // page, -(-length // page)))
    cache = random_cache(g, pages, 2, page, dim)
    cache[1].copy_((cache[1].float() * 2.0 ** -max(-110, min(exponent, 118))).to(torch.bfloat16))
    q = (torch.randn((news, 8, dim), generator=g, device="cuda").clamp(-1.9, 1.9) * 2.0 ** exponent).to(torch.bfloat16)
    q[0, 0] = 0
    args = (table, ints([length]), begins([news]))
    got = ops.cache_attention(q, cache, *args).double()
    want, bound = expected(q, cache, table, length, news, dim ** -0.5)
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())
    ops.check_device_error()


@pytest.mark.parametrize("dim,news,room", CASES)
def test_keys_and_scores_near_the_largest_float(ops, dim, news, room):  # noqa: F811
    g = generator(dim + news)
    length = 300
    for top, q_value in ((2.0 ** 112, 1.0), (2.0 ** 112, 2.0 ** -100), (2.0 ** -8, 1.5 * 2.0 ** 120)):
        keys = top * torch.randint(-8, 9, (length,), generator=g, device="cuda").float()
        run(ops, g, dim, news, room, length, keys, q_value, scale=2.0 ** -5)
        run(ops, g, dim, news, room, length, keys, -q_value)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim,news,room", CASES)
@pytest.mark.parametrize("exponent", [4, 8, 12, 14])
@pytest.mark.parametrize("at", [2, 3, 60])
def test_a_large_dimension_of_queries_where_keys_are_zero(ops, dim, news, room, exponent, at, kind):  # noqa: F811
    """It has no part in the scores, and takes no place from those that have: they are sums in f32."""
    g = generator(dim + exponent)
    length, page = 512, 64
    pages, table = layout(g, [length], page, width=max(room // page, -(-length // page)))
    cache = random_cache(g, pages, 2, page, dim)
    keys, step = cache[0], cache[1][..., :1].float()
    cache[1][..., 1:] = (-8 * step).to(torch.bfloat16)   # code 8 is zero
    keys[..., at // 2] = (keys[..., at // 2] & 0xF0) | 0x08 if at % 2 == 0 else (keys[..., at // 2] & 0x0F) | 0x80
    q = torch.randn((news, 8, dim), generator=g, device="cuda")
    q[..., at] = 2.0 ** exponent
    q = q.to(TYPES[kind])
    args = (table, ints([length]), begins([news]))
    got = ops.cache_attention(q, cache, *args).double()
    # Without that dimension the same tokens are as far from 64 bits as the kernel's roundings take them.  With it the other dimensions are
    # f16 numbers down to 2^-35 of it, 2^-21 at most: no more than a hundredth of an output's rounding.
    blank = q.clone()
    blank[..., at] = 0
    want = expected(blank, cache, table, length, news, dim ** -0.5)[0]
    usual = (ops.cache_attention(blank, cache, *args).double() - want).norm()
    assert float((got - want).norm() / usual) <= 1.25, float((got - want).norm() / usual)


@pytest.mark.parametrize("dim,news,room", CASES)
@pytest.mark.parametrize("which", [0, 1, 2])
def test_steps_below_zero(ops, dim, news, room, which):  # noqa: F811
    """A cache that another program has filled: a code stands for least + step * code whatever the step's sign."""
    g = generator(dim + news)
    length, page = 400, 64
    pages, table = layout(g, [length], page, width=max(room // page, -(-length // page)))
    cache = random_cache(g, pages, 2, page, dim)
    plain = [t.clone() for t in cache]
    flip = torch.rand(cache[1].shape[:3], generator=g, device="cuda") < (0.0, 0.5, 1.0)[which]
    for i in (0, 2):   # the same values: codes from the other end, least + 15 step and -step
        cache[i][flip] = 255 - cache[i][flip]
        step, least = cache[i + 1][..., 0].float(), cache[i + 1][..., 1].float()
        step = (step * 8).ceil() / 8   # (numbers whose multiples by 15 bf16 holds)
        least = (least * 2).round() / 2
        for to, sign in ((plain, 1.0), (cache, -1.0)):
            to[i + 1][..., 0] = torch.where(flip, sign * step, step).to(torch.bfloat16)
            to[i + 1][..., 1] = torch.where(flip, least + (15 * step if sign < 0 else 0), least).to(torch.bfloat16)
    for i in (0, 2):
        (ca, sa, la), (cb, sb, lb) = (R.rows_of(c[i], c[i + 1]) for c in (plain, cache))
        assert torch.equal(ca * sa + la, cb * sb + lb)
    q = torch.randn((news, 8, dim), generator=g, device="cuda").to(torch.float16)
    args = (table, ints([length]), begins([news]))
    got = ops.cache_attention(q, cache, *args).double()
    want, bound = expected(q, plain, table, length, news, dim ** -0.5)
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())
    ops.check_device_error()
