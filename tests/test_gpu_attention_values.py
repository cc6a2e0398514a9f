"""Values whose steps are far from their neighbours', seen by some queries of a piece and not by others."""
import math

import pytest
import torch

from tests import cache_reference as R
from tests.test_gpu_cache import begins, generator, ints, layout, ops, random_cache  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("per,news", [(4, 20), (1, 20), (32, 9), (4, 300)])
@pytest.mark.parametrize("step", [2.0 ** 40, 2.0 ** 110, math.inf])
def test_large_steps_that_some_queries_do_not_see(ops, dim, per, news, step):  # noqa: F811
    g = generator(1)
    length = news + 30
    pages, table = layout(g, [length], 16)
    cache = random_cache(g, pages, 2, 16, dim)
    q = torch.randn((news, 2 * per, dim), generator=g, device="cuda").to(torch.bfloat16)
    args = (table, ints([length]), begins([news]))
    blank = torch.zeros_like(q)
    want, bound = R.attention(q, cache, *args, dim ** -0.5, blank)
    at = length - 5   # the last five queries see it
    cache[3][int(table[0, at // 16]), :, at % 16, 0] = step
    got = ops.cache_attention(q, cache, *args).double()
    assert bool(((got - want).abs()[:-5] <= bound[:-5]).all())
    if step < 2.0 ** 100:
        want, bound = R.attention(q, cache, *args, dim ** -0.5, blank)
        # A term enters as p step (code - 8) beside p (least + 8 step): its rounding to f16 is off by up to 8 p step 2^-11, whatever
        # the code is, where the bound counts code p step 2^-11; and up to 400 f32 additions of 8 p step are off by 400 * 8 * 2^-23 < 2^-11
        # of p step.  sum p step is what attention gives for codes of 1 and least values of 0.
        ones = cache._replace(v=torch.full_like(cache.v, 0x11), v_scale=torch.cat((cache.v_scale[..., :1], torch.zeros_like(cache.v_scale[..., :1])), -1))
        bound += 9 * 2.0 ** -11 * R.attention(q, ones, *args, dim ** -0.5, blank)[0]
        # p step enters as f16 times a power of two that takes the largest step to 64 or more, so that f16's finest step, 2^-24, is
        # 2^-30 of that step: terms of tiny p are off by half of it, times 8 (and a sum of p is 1 at least, the reference being one).
        bound += length * 8 * 2.0 ** -31 * step
        assert bool(((got - want).abs() <= bound).all())
    ops.check_device_error()
