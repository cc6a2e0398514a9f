"""Which kernel a product runs on: rules that hold for every tile variant, split and list of groups.  No GPU needed."""
import random

import pytest

from ptq_int8_lab_b200 import engine as E
from ptq_int8_lab_b200 import ops as O

GROUPS = (0, 1, 2, 8, 31, 200, 777, 1024)


def every_launch():
    """Each variant with each split that it takes, for one group and for lists of all lengths."""
    for v in range(O.linear_variants()):
        for split in (1, 2, 4, 8):
            for groups in GROUPS:
                for bits in (8, 4):
                    for act in (O.EPI_NONE, O.EPI_SWIGLU):
                        c = O.linear_choice(5000, 4096, 1024, bits, act, groups, variant=v, split=split)
                        if c:
                            yield v, split, groups, c


def test_stages_are_multiples_of_the_turns():
    """Unpacking sets take turns at the stages and at the operand tiles; a barrier's parity tells two phases apart, so each
    has to belong to one set."""
    seen = set()
    for v, split, groups, c in every_launch():
        assert c.variant == v and c.split == split
        assert c.stages % c.turns == 0 and c.operand_tiles % c.turns == 0, c
        assert 2 <= c.stages <= 12 and c.operand_tiles <= c.stages, c
        assert (c.operand_tiles > 0) == (c.w_bits == 4)
        seen.add(v)
    assert seen == set(range(O.linear_variants()))


def test_shared_memory_keeps_tmem_apart():
    """CTAs that share an SM take half of its TMEM columns each, so three of them must not fit; the others take all of
    them, so none of them may stand beside another.  1 KB of each CTA is the system's."""
    sizes = {c.smem_bytes for *_, c in every_launch()}
    two, one = {s for s in sizes if s <= 113 * 1024}, {s for s in sizes if s > 113 * 1024}
    assert two and one and max(one) <= 227 * 1024
    assert 3 * (min(two) + 1024) > 228 * 1024 >= 2 * (max(two) + 1024)
    assert min(one) + min(two) + 2048 > 228 * 1024


def test_some_variant_serves_every_call():
    rng = random.Random(0)
    for _ in range(3000):
        rows, k, n = (int(2 ** rng.uniform(0, top)) for top in (14, 17, 15))
        groups, bits, act = rng.choice(GROUPS), rng.choice((8, 4)), rng.choice((0, 1))
        c = O.linear_choice(rows, min(k, 131071), n, bits, act, groups)
        assert c.kernel in (O.KERNEL_FEW, O.KERNEL_TILES)
        if c.kernel == O.KERNEL_TILES:
            assert (c.w_bits, c.epilogue) == (bits, act)
            assert O.linear_choice(rows, min(k, 131071), n, bits, act, groups, variant=c.variant, split=c.split) == c


def test_layouts_that_no_tile_can_read():
    for rows, k, n, bits, kernel in ((20, 1001, 64, 8, O.KERNEL_ANY), (20, 1001, 64, 4, O.KERNEL_ANY), (20, 1008, 64, 8, O.KERNEL_TILES),
                                     (1, 1001, 1, 8, O.KERNEL_TILES), (1, 1001, 2, 8, O.KERNEL_ANY), (2, 1024, 64, 4, O.KERNEL_FEW)):
        assert O.linear_choice(rows, k, n, bits, pitch=1).kernel == kernel


@pytest.mark.parametrize("variant,split", [(0, 3), (0, 16), (0, 0), (0, -1), (19, 2), (10 ** 6, 1)])
def test_what_no_variant_takes(variant, split):
    assert O.linear_choice(500, 4096, 1024, variant=variant, split=split) is None


def test_refusals():
    for bad in (dict(rows=0, in_features=64, out_features=8), dict(rows=1, in_features=131072, out_features=8),
                dict(rows=1, in_features=64, out_features=8, bits=3), dict(rows=4, in_features=64, out_features=8, groups=1025)):
        with pytest.raises(E.Ptq8Error):
            O.linear_choice(**bad)
    assert E.lib().ptq8_linear_choose(148, None, 0, None) == 1 and E.lib().ptq8_linear_choose_as(148, None, 0, 0, 1, None) == 1
    assert E.lib().ptq8_ops_set_choice_test(None, 0, 1) == 1


def test_weights_that_the_few_token_kernel_takes():
    """Up to 18 MB of weights, 24 MB for one token on int4 codes: above, tiles were faster (4096 x 5632 int8 from DRAM:
    9.9 and 7.4 us)."""
    few, tiles = O.KERNEL_FEW, O.KERNEL_TILES
    for rows in (1, 2, 4):
        for act in (0, 1):
            for n, kernel in ((4096, few), (4608, few), (4624, tiles), (5632, tiles), (8192, tiles)):
                assert O.linear_choice(rows, 4096, n // (1 + act), 8, act).kernel == kernel
            for n, kernel in ((9216, few), (9248, few if rows == 1 else tiles), (12288, few if rows == 1 else tiles), (12320, tiles)):
                assert O.linear_choice(rows, 4096, n // (1 + act), 4, act).kernel == kernel
    assert O.linear_choice(5, 4096, 64).kernel == tiles and O.linear_choice(4, 4096, 64).kernel == few
    assert O.linear_choice(8, 1024, 1024, groups=8).kernel == few and O.linear_choice(9, 1024, 1024, groups=8).kernel == tiles
