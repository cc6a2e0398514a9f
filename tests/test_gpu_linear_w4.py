"""Products of float activations with 4-bit weights in groups, against 64 bits."""
import math

import pytest
import torch

from ptq_int8_lab_b200 import engine as E

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    from ptq_int8_lab_b200.ops import Int8Ops
    with Int8Ops(0) as o:
        yield o


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def weights(g, channels, inp, group, scale_type="f32", pitch=16):
    wide = (inp + 1) // 2
    w = torch.randint(0, 256, (channels, -(-wide // pitch) * pitch), generator=g, device="cuda").to(torch.uint8)[:, :wide]
    s = (torch.rand((channels, -(-inp // group)), generator=g, device="cuda") * 0.02 + 0.002).to(TYPES[scale_type])
    return w, s


def expected(x, w, s, group, bias, gated, out_type):
    """(y, bound) in 64 bits.  A sum is of f32 additions of terms (code + 8) x and -8 x, 16 at a time, then of a group's sum times
    its scale: at most (40 + groups) roundings of 2^-23 (or cuts of as much) of the terms' magnitudes, or in / 64 + 10 where single
    products are added; f32 activations keep 22 places."""
    inp = x.shape[1]
    c = torch.stack((w & 15, w >> 4), -1).flatten(1)[:, :inp].double()
    c = torch.where(c > 7, c - 16, c)
    scale = s.double().repeat_interleave(group, 1)[:, :inp]
    y = x.double() @ (c * scale).t()
    size = x.double().abs() @ ((c.abs() + 16) * scale.abs()).t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    bound = size * 2.0 ** -23 * (max(40 + s.shape[1], inp / 64 + 10) + 2)
    if gated:
        n = y.shape[1] // 2
        a, u, ba, bu = y[:, :n], y[:, n:], bound[:, :n], bound[:, n:]
        act = torch.nn.functional.silu(a)
        y, bound = act * u, 1.1 * ba * u.abs() + act.abs() * bu + ba * bu + (act * u).abs() * 2.0 ** -20
    half = torch.finfo(out_type).eps / 2
    return y, bound * (1 + half) + half * y.abs() + (2.0 ** -25 if out_type == torch.float16 else 2.0 ** -130)


def check(ops, g, tokens, inp, out, group, x_type="bf16", out_type="bf16", scale_type="f32", gated=False, bias=False, pitch=16, x=None):
    from ptq_int8_lab_b200.ops import EPI_NONE, EPI_SWIGLU
    channels = out * (2 if gated else 1)
    w, s = weights(g, channels, inp, group, scale_type, pitch)
    if x is None:
        x = (torch.randn((tokens, inp), generator=g, device="cuda") * (torch.rand((tokens, 1), generator=g, device="cuda") + 0.1)).to(TYPES[x_type])
    b = torch.randn(channels, generator=g, device="cuda") if bias else None
    got = ops.linear_w4(x, w, s, group, bias=b, act=EPI_SWIGLU if gated else EPI_NONE, dtype=TYPES[out_type])
    want, bound = expected(x, w, s, group, b, gated, TYPES[out_type])
    assert got.dtype == TYPES[out_type] and got.shape == want.shape
    worst = float(((got.double() - want).abs() / bound).max())
    assert worst <= 1.0, worst
    return got


@pytest.mark.parametrize("x_type", list(TYPES))
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 70])
def test_tokens_and_groups(ops, x_type, group, tokens):
    check(ops, generator(tokens + group), tokens, 1024, 160, group, x_type, out_type="f32")


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("x_type,out_type,scale_type", [("bf16", "bf16", "f16"), ("f16", "f32", "bf16"), ("f32", "f16", "f32")])
@pytest.mark.parametrize("inp,out,group", [(1, 1, 32), (31, 5, 32), (33, 17, 32), (127, 16, 64), (130, 8, 128), (2000, 1270, 32), (257, 33, 257),
                                           (4096, 40, 128), (1100, 24, 64), (96, 7, 1000)])
def test_odd_sizes(ops, inp, out, group, x_type, out_type, scale_type, gated):
    for tokens in (1, 7, 12):
        check(ops, generator(inp + out), tokens, inp, out, group, x_type, out_type, scale_type, gated, bias=True)


@pytest.mark.parametrize("group", [1, 7, 16, 48, 100])
@pytest.mark.parametrize("x_type", list(TYPES))
def test_any_group(ops, group, x_type):
    check(ops, generator(group), 5, 333, 40, group, x_type, "f32", gated=True, bias=True)


@pytest.mark.parametrize("out", [3, 7000, 20000])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("x_type", ["f32", "bf16"])
def test_many_channels(ops, out, gated, x_type):
    """One, two and four tiles of rows a warp."""
    for group in (32, 128):
        check(ops, generator(out), 6, 384, out, group, x_type, gated=gated)


@pytest.mark.parametrize("pitch", [1, 2, 4, 8, 32])
def test_layouts(ops, pitch):
    """Weights at any byte, activations and outputs at any element: the same values (one kernel or the other)."""
    for group in (32, 64, 128):
        check(ops, generator(pitch), 3, 650, 50, group, "f16", "f32", pitch=pitch)
    g = generator(pitch)
    w, s = weights(g, 48, 512, 64)
    x = torch.randn((5, 512), generator=g, device="cuda").to(torch.bfloat16)
    want = ops.linear_w4(x, w, s, 64)
    for off in (1, 3, 8):
        wide = torch.zeros((5, 531), dtype=torch.bfloat16, device="cuda")
        wide[:, off:off + 512] = x
        out = torch.full((5, 60), 9.0, dtype=torch.bfloat16, device="cuda")
        ops.linear_w4(wide[:, off:off + 512], w, s, 64, out=out[:, off:off + 48])
        assert torch.equal(out[:, off:off + 48], want) and (out[:, :off] == 9).all() and (out[:, off + 48:] == 9).all()
        ops.linear_w4(x, w, torch.cat((s, s), 1)[:, :s.shape[1]], 64, out=out[:, :48])
        assert torch.equal(out[:, :48], want)


def test_the_last_row_ends_the_allocation(ops):
    """Weights whose last row ends where its tensor ends, without the pitch's rest: nothing behind it is read for its value."""
    g = generator(2)
    w, s = weights(g, 32, 1000, 128)
    flat = torch.zeros(31 * 512 + 500, dtype=torch.uint8, device="cuda")
    tight = flat.as_strided((32, 500), (512, 1))
    tight.copy_(w)
    x = torch.randn((2, 1000), generator=g, device="cuda")
    assert torch.equal(ops.linear_w4(x, tight, s, 128), ops.linear_w4(x, w, s, 128))


@pytest.mark.parametrize("x_type", list(TYPES))
def test_sizes_far_apart(ops, x_type):
    """Outliers, tiny tokens, zero tokens, large ones: each keeps its own scale."""
    g = generator(7)
    x = torch.randn((8, 1024), generator=g, device="cuda")
    small, large = (2.0 ** -14, 1000.0) if x_type == "f16" else (2.0 ** -60, 2.0 ** 60)
    x[0] *= small
    x[1] *= large
    x[2] = 0
    x[3, ::128] *= 1000
    check(ops, g, 8, 1024, 64, 64, x_type, "f32", x=x.to(TYPES[x_type]))


@pytest.mark.parametrize("x_type", list(TYPES))
def test_tokens_that_are_not_finite(ops, x_type):
    """NaN for that token, nothing for the others."""
    g = generator(8)
    w, s = weights(g, 40, 512, 64)
    x = torch.randn((6, 512), generator=g, device="cuda").to(TYPES[x_type])
    good = ops.linear_w4(x, w, s, 64)
    x[1, 5], x[3, 500], x[4, 0] = math.nan, math.inf, -math.inf
    got = ops.linear_w4(x, w, s, 64)
    assert torch.isnan(got[[1, 3, 4]]).all() and torch.equal(got[[0, 2, 5]], good[[0, 2, 5]])


def test_no_tokens(ops):
    w, s = weights(generator(9), 40, 512, 64)
    assert ops.linear_w4(torch.empty((0, 512), device="cuda"), w, s, 64).shape == (0, 40)


def test_the_same_twice(ops):
    g = generator(10)
    w, s = weights(g, 512, 2048, 64)
    x = torch.randn((8, 2048), generator=g, device="cuda").to(torch.bfloat16)
    first = ops.linear_w4(x, w, s, 64)
    assert all(torch.equal(ops.linear_w4(x, w, s, 64), first) for _ in range(20))


def test_refusals(ops):
    from ptq_int8_lab_b200.ops import EPI_SWIGLU
    w, s = weights(generator(11), 40, 512, 64)
    x = torch.zeros((2, 512), device="cuda")
    for change, text in ((dict(group=0), "group"), (dict(group=32), "w_scale"), (dict(x=x.cpu()), "cpu"), (dict(x=x.double()), "dtype"),
                         (dict(x=x[:, :510]), "rows of"), (dict(w=w.to(torch.int32)), "dtype"), (dict(w_scale=s[:, :7]), "w_scale"),
                         (dict(bias=torch.zeros(39, device="cuda")), "bias"), (dict(act=2), "act"), (dict(dtype=torch.float64), "dtype"),
                         (dict(out=torch.zeros((2, 41), device="cuda")), "out"), (dict(x=x.t()), "x"), (dict(stream=torch.cuda.current_stream()), "out"),
                         (dict(w=w[:39], w_scale=s[:39], act=EPI_SWIGLU), "gate")):
        args = dict(x=x, w=w, w_scale=s, group=64)
        args.update(change)
        with pytest.raises(E.Ptq8Error, match=text):
            ops.linear_w4(**args)
