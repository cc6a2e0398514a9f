"""linear_w4 where shared memory does not hold all activations: they are brought in a segment of 16 x 128 features at a time.

A block has 224 KB: 16 KB for sums, 64 KB for a stage of weights, and 2080 bytes for 128 features of eight columns (a token each, two for
f32): 70 x 128 features of eight tokens fit, 140 x 128 of four."""
import pytest
import torch

from ptq_int8_lab_b200 import engine as E
from tests.test_gpu_linear_w4 import TYPES, check, generator, ops, weights  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x_type", list(TYPES))
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("inp,group", [(9000, 32), (9216, 64), (14336, 128), (16400, 32), (10240, 10240)])
def test_long_rows(ops, inp, group, gated, x_type):  # noqa: F811
    """Last segments of fewer chunks than warps share a tile, widths that end inside a chunk, one pass of tokens and several."""
    for tokens in (8, 13, 40):
        check(ops, generator(inp + tokens), tokens, inp, 72, group, x_type, "f32" if gated else "bf16", "f16", gated=gated, bias=True)


@pytest.mark.parametrize("x_type", list(TYPES))
@pytest.mark.parametrize("out", [1, 5000, 40000])
def test_many_channels(ops, out, x_type):  # noqa: F811
    """From one tile that all warps share to several rounds of tiles a warp, with a second pass of tokens."""
    check(ops, generator(out), 11, 9100, out, 64, x_type, "bf16", "f16")


def test_rounds_of_gated_tiles(ops):  # noqa: F811
    check(ops, generator(5), 8, 9728, 30000, 128, "bf16", "bf16", "f16", gated=True)


def test_the_same_twice(ops):  # noqa: F811
    g = generator(6)
    w, s = weights(g, 3000, 14336, 128)
    x = torch.randn((16, 14336), generator=g, device="cuda").to(torch.bfloat16)
    first = ops.linear_w4(x, w, s, 128)
    assert all(torch.equal(ops.linear_w4(x, w, s, 128), first) for _ in range(20))
    ops.check_device_error()


@pytest.mark.parametrize("x_type", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,out,gated", [(8, 64, False), (21, 5000, True)])
def test_a_wait_runs_out(tokens, out, gated, x_type):
    from ptq_int8_lab_b200.ops import EPI_NONE, EPI_SWIGLU, Int8Ops
    with Int8Ops(0) as own:
        g = generator(7)
        w, s = weights(g, out * (2 if gated else 1), 14336, 64)
        x = torch.randn((tokens, 14336), generator=g, device="cuda").to(TYPES[x_type])
        args = dict(act=EPI_SWIGLU if gated else EPI_NONE)
        good = own.linear_w4(x, w, s, 64, **args)
        own.check_device_error()
        own.set_wait_test(10_000_000, True)
        own.linear_w4(x, w, s, 64, **args)
        with pytest.raises(E.Ptq8Error, match="ran out") as e:
            own.check_device_error()
        assert e.value.status == 4
        own.set_wait_test()
        assert torch.equal(own.linear_w4(x, w, s, 64, **args), good)
        own.check_device_error()
