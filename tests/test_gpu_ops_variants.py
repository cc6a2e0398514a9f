"""Every tile variant of the tensor-core product with every split, one weight matrix or groups, whatever a call of that
size would choose: outputs against plain 64-bit forms."""
import numpy as np
import pytest
import torch
from test_gpu_ops import case, check, dev, laid, pack4, plain_grouped, plain_product

from ptq_int8_lab_b200 import engine as E
from ptq_int8_lab_b200 import ops as O

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ops():
    return O.Int8Ops(0)


def launches():
    for v in range(O.linear_variants()):
        for split in (1, 2, 4, 8):
            c = [O.linear_choice(500, 4096, 1024, bits, act, variant=v, split=split) for bits in (8, 4) for act in (0, 1)]
            for one in filter(None, c):
                yield pytest.param(one, id=f"{one.ctas}x{one.tokens}-int{one.w_bits}{'-gated' if one.epilogue else ''}-split{split}")


@pytest.mark.parametrize("c", list(launches()))
@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("k,n", [(1100, 300), (8199, 130), (2048, 1025)])
def test_variant(ops, c, grouped, k, n):
    """Input features that end inside a block, channels that end inside a tile; rows of less than a tile, and of a few
    tiles and a part; more stages than there are, so that barriers come round."""
    rng = np.random.default_rng(c.variant * 8 + c.split)
    gated, bits = bool(c.epilogue), c.w_bits
    for counts in ([1], [c.tokens + 5], [2 * c.tokens + 17]) if not grouped else ([3, 0, c.tokens + 1, 1, 2 * c.tokens, 17],):
        rows, groups = sum(counts), len(counts) if grouped else 0
        x, xs, w, ws, b = case(rng, rows, k, n, bits, gated, True, groups)
        wd = laid(w if bits == 8 else pack4(w))
        ops.set_choice_test(c.variant, c.split)
        if grouped:
            offs = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
            a = (laid(x), dev(xs), dev(offs), wd, dev(ws), dev(b))
            check(lambda t: ops.linear_grouped(*a, bits=bits, act=c.epilogue, dtype=t), plain_grouped(x, xs, offs, w, ws, b), n, gated, "f32")
        else:
            a = (laid(x), dev(xs), wd, dev(ws), dev(b))
            check(lambda t: ops.linear(*a, bits=bits, act=c.epilogue, dtype=t), plain_product(x, xs, w, ws, b), n, gated, "bf16")
    ops.check_device_error()


@pytest.mark.parametrize("c", list(launches()))
def test_many_tiles(ops, c):
    """More tiles than the device runs at once: every CTA takes several, and a split's clusters come in waves."""
    rng = np.random.default_rng(c.variant)
    gated, bits = bool(c.epilogue), c.w_bits
    rows, n = 3 * c.tokens + 1, 128 * c.ctas * 148 // c.split // 2 + 70
    k = 128 * c.split * 2 + 40
    x, xs, w, ws, b = case(rng, rows, k, n, bits, gated, True)
    a = (laid(x), dev(xs), laid(w if bits == 8 else pack4(w)), dev(ws), dev(b))
    ops.set_choice_test(c.variant, c.split)
    check(lambda t: ops.linear(*a, bits=bits, act=c.epilogue, dtype=t), plain_product(x, xs, w, ws, b), n, gated, "f32")
    ops.check_device_error()


@pytest.mark.parametrize("c", list(launches()))
@pytest.mark.parametrize("grouped", [False, True])
def test_wait_runs_out(ops, c, grouped):
    """The first load never comes: the launch gives up, reports it, and the next one is right."""
    rng = np.random.default_rng(1)
    rows, k, n = 2 * c.tokens + 1, 1024, 600
    x, xs, w, ws, _ = case(rng, rows, k, n, c.w_bits, bool(c.epilogue), False, 2 if grouped else 0)
    a = [laid(x), dev(xs), laid(w if c.w_bits == 8 else pack4(w)), dev(ws)]
    if grouped:
        a.insert(2, torch.tensor([0, c.tokens + 1, rows], dtype=torch.int32, device="cuda"))
    call = ops.linear_grouped if grouped else ops.linear
    ops.set_choice_test(c.variant, c.split)
    good = call(*a, bits=c.w_bits, act=c.epilogue)
    ops.check_device_error()
    ops.set_wait_test(3_000_000, True)
    call(*a, bits=c.w_bits, act=c.epilogue)
    with pytest.raises(E.Ptq8Error, match="ran out"):
        ops.check_device_error()
    ops.set_wait_test()
    assert torch.equal(call(*a, bits=c.w_bits, act=c.epilogue), good)
    ops.check_device_error()


def test_refusals(ops):
    a = (torch.zeros((9, 64), dtype=torch.int8, device="cuda"), torch.ones(9, device="cuda"),
         torch.zeros((32, 64), dtype=torch.int8, device="cuda"), torch.ones(32, device="cuda"))
    with pytest.raises(E.Ptq8Error, match="variant 1000"):
        ops.set_choice_test(1000)
    int4 = next(v for v in range(O.linear_variants()) if O.linear_choice(9, 64, 32, 4, variant=v))
    for variant, split in ((int4, 1), (0, 3), (0, 2)):   # another weight type, no such split, more CTAs than blocks
        ops.set_choice_test(variant, split)
        with pytest.raises(E.Ptq8Error, match="does not serve"):
            ops.linear(*a)
    ops.set_choice_test(0)
    with pytest.raises(E.Ptq8Error, match="this layout"):
        ops.linear(torch.zeros((9, 65), dtype=torch.int8, device="cuda")[:, :64], *a[1:])
    ops.set_choice_test()
    ops.linear(*a)
    ops.check_device_error()
