"""linear_w4 where one activation is far larger than those beside it and meets codes of zero: the others' outputs keep f32's accuracy."""
import pytest
import torch

from tests.test_gpu_linear_w4 import TYPES, generator, ops, weights  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


def expected(x, w, s, group, out_type):
    """(y, bound) in 64 bits.  Of 128 activations that begin at a multiple of 128 the largest, `top`, becomes 2^14 .. 2^15; f16 numbers are
    multiples of 2^-24 there, so one is off by at most 2^-39 top, or 2^-35 top where its index is odd (it enters as a sixteenth).  f32
    ones enter as two f16: off by 2^-22 of themselves too.  Sums: at most (40 + groups) or (in / 64 + 10) roundings of 2^-23, or cuts of as
    much, of the terms' magnitudes; the tensor cores may take a zero's exponent for 2^-14, which counts as a term of 2^-14 top in each
    product of 16."""
    tokens, inp = x.shape
    c = torch.stack((w & 15, w >> 4), -1).flatten(1)[:, :inp].double()
    c = torch.where(c > 7, c - 16, c)
    scale = s.double().repeat_interleave(group, 1)[:, :inp]
    y = x.double() @ (c * scale).t()
    top = x.double().abs().view(tokens, -1, 128).amax(-1).repeat_interleave(128, 1)
    grain = top * torch.tensor([2.0 ** -39, 2.0 ** -35], dtype=torch.float64, device="cuda").repeat(inp // 2)
    if x.dtype == torch.float32:
        grain = grain + x.double().abs() * 2.0 ** -22
    size = x.double().abs() @ (c.abs() * scale).t() + 2.0 ** -14 / 16 * top @ scale.t()
    bound = grain @ (c.abs() * scale).t() + size * 2.0 ** -23 * (max(40 + s.shape[1], inp / 64 + 10) + 2)
    half = torch.finfo(out_type).eps / 2
    return y, bound * (1 + half) + half * y.abs() + (2.0 ** -25 if out_type == torch.float16 else 2.0 ** -130)


@pytest.mark.parametrize("x_type", list(TYPES))
@pytest.mark.parametrize("out_type", list(TYPES))
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens", [1, 2, 3, 8, 20, 40])
def test_outliers_beside_codes_of_zero(ops, tokens, group, x_type, out_type):  # noqa: F811
    g = generator(tokens + group)
    inp = 1024
    for exponent in (4, 8, 12, 16) + (() if x_type == "f16" else (22, 30)):
        for at in (2, 3, 640, 1021):
            w, s = weights(g, 48, inp, group)
            w[:, at // 2] = w[:, at // 2] & (0xF0 if at % 2 == 0 else 0x0F)   # code 0
            x = torch.randn((tokens, inp), generator=g, device="cuda")
            x[:, at] = 0.99 * 2.0 ** exponent
            x = x.to(TYPES[x_type])
            y = ops.linear_w4(x, w, s, group, dtype=TYPES[out_type]).double()
            want, bound = expected(x, w, s, group, TYPES[out_type])
            worst = float(((y - want).abs() / bound).max())
            assert worst <= 1.0, (exponent, at, worst)


@pytest.mark.parametrize("x_type", ["f16", "bf16"])
@pytest.mark.parametrize("at", [0, 1])
def test_activations_within_a_range_are_exact(ops, at, x_type):  # noqa: F811
    """16-bit activations within 2^-24 of the largest among 128 lose nothing: one of them alone meets a code of one."""
    g = generator(at)
    inp = 256
    for below in (0, 10, 20, 23):
        x = torch.zeros((8, inp), device="cuda")
        x[:, 6] = 2.0 ** 8
        x[:, 130] = 1.0
        x[:, 32 + at] = (torch.rand(8, generator=g, device="cuda") + 1.0) * 2.0 ** (8 - below - 1)
        x = x.to(TYPES[x_type])
        w = torch.zeros((16, inp // 2), dtype=torch.uint8, device="cuda")
        w[:, 16] = 16 if at else 1
        y = ops.linear_w4(x, w, torch.ones((16, 2), device="cuda"), 128, dtype=torch.float32)
        assert torch.equal(y, x[:, 32 + at:33 + at].float().expand(8, 16))
