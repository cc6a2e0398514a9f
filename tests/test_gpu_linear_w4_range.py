"""linear_w4 over the whole range of its activations, on each of its kernels, against 64 bits."""
import pytest
import torch

from tests.test_gpu_linear_w4 import TYPES, check, expected, generator, ops, weights  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x_type,out_type", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("group,pitch", [(32, 16), (64, 16), (128, 16), (64, 1), (24, 16)])
@pytest.mark.parametrize("tokens", [1, 2, 3, 8, 21])
def test_the_largest_floats(ops, tokens, group, pitch, x_type, out_type):  # noqa: F811
    """Activations up to the type's largest, alone in their groups or all of a size: finite outputs are as near as any."""
    g = generator(tokens)
    x = torch.randn((tokens, 1024), generator=g, device="cuda").clamp(-4, 4)
    for t in range(tokens):
        x[t] *= 2.0 ** (113, 116, 119, 0)[t % 4]
    x[tokens - 1, ::200] = 1.5 * 2.0 ** 117
    x[0, 77] = 1.75 * 2.0 ** 127   # (an odd feature; times a scale of at most 0.022 and a code of 8)
    x[0, 500] = -1.25 * 2.0 ** 126
    check(ops, g, tokens, 1024, 200, group, x_type, out_type, pitch=pitch, x=x.to(TYPES[x_type]))


@pytest.mark.parametrize("x_type", ["f32", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens", [1, 3, 8, 21])
def test_small_floats(ops, tokens, group, x_type):  # noqa: F811
    """Down to 2^-100 as the largest of 128, and (with what is documented) below."""
    g = generator(group + tokens)
    x = torch.randn((tokens, 512), generator=g, device="cuda")
    x[:, ::128] = 2.0   # the largest is 2^-99 at least
    check(ops, g, tokens, 512, 48, group, x_type, "f32", x=(x * 2.0 ** -100).to(TYPES[x_type]))
    w, s = weights(g, 48, 512, group)
    for e in (-112, -126):
        x = (torch.randn((tokens, 512), generator=g, device="cuda") * 2.0 ** e).to(TYPES[x_type])
        y = ops.linear_w4(x, w, s, group, dtype=torch.float32).double()
        want, bound = expected(x, w, s, group, None, False, torch.float32)
        # activations enter as multiples of 2^-24 after 2^114 (odd features 2^-20): off by half of that, 2^-135, times codes of 8 at most;
        # sums are kept in units of 2^12 at most, whose finest number is 2^-149: 16 sums a group or feature are off by 2^-137 each
        grain = 8 * 2.0 ** -135 * s.double().repeat_interleave(group, 1)[:, :512].sum(1) + 512 * 2.0 ** -137
        assert bool(((y - want).abs() <= bound + grain).all())


def test_outputs_past_a_float(ops):  # noqa: F811
    """What no f32 number holds is infinite, and of the right sign."""
    g = generator(3)
    w = torch.full((40, 128), 0x77, dtype=torch.uint8, device="cuda")
    s = torch.ones((40, 2), device="cuda")
    for tokens in (1, 3, 8):
        x = torch.full((tokens, 256), 2.0 ** 126, device="cuda")
        x[-1] *= -1
        x[0, 0] *= torch.rand((), generator=g, device="cuda") + 0.5
        y = ops.linear_w4(x, w, s, 128)
        assert bool(torch.isinf(y).all()) and bool((y[-1] < 0).all()) and (tokens == 1 or bool((y[0] > 0).all()))
    ops.check_device_error()
