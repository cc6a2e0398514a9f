"""quantize_rows with much to read: the kernels that hold two and four vectors a thread, several rows in a block, and last
blocks with rows missing.  Against the definition in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MANY = 1 << 20   # vectors of 16 bytes from which a call counts as large


@pytest.fixture(scope="module")
def ops():
    from ptq_int8_lab_b200.ops import Int8Ops
    return Int8Ops(0)


def plain(x):
    """(codes, scale): the scale's two 32-bit steps, then the quotient in 64 bits (float64 division of two floats rounds to
    a half only where the exact quotient is one: it has at most 48 bits)."""
    top = x.float().abs().amax(1)
    scale = (top / torch.full_like(top, 127.0)).clamp_min(1e-8)
    q = x.double() / scale.double()[:, None]
    return ((q.abs() + 0.5).floor() * q.sign()).to(torch.int8), scale


def made(rows, width, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, width), generator=g, device="cuda")
    x[::7] *= 31
    x[3::11, ::2] = 0
    x[min(5, rows - 1)] = 0
    return x.to(DT[dtype])


# vectors a row holds: one for each kernel of the large calls, at both ends of its range, and the longest rows
VECS = [1, 32, 33, 64, 65, 128, 129, 256, 257, 512, 513, 1024, 1025, 2048, 2049, 4096, 4097]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vecs", VECS)
@pytest.mark.parametrize("layout", ["plain", "odd width", "odd start"])
def test_large(ops, dtype, vecs, layout):
    lanes = 4 if dtype == "f32" else 8
    rows = MANY // vecs + 3   # odd or even, never a whole number of blocks
    rows += rows % 4 == 0
    width = vecs * lanes - (1 if layout == "odd width" else 0)
    x = made(rows, width, dtype, vecs)
    if layout == "odd start":
        buf = torch.empty(rows * width + 3, dtype=DT[dtype], device="cuda")
        buf[3:].view(rows, width).copy_(x)
        x = buf[3:].view(rows, width)
    codes, scale = ops.quantize_rows(x)
    want, s = plain(x)
    assert torch.equal(scale, s)
    assert torch.equal(codes, want)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("width", [250, 256, 520, 1000, 2048, 4104, 8191])
def test_large_gathers(ops, dtype, width):
    """More rows out than in, some of indices that are no rows."""
    lanes = 4 if dtype == "f32" else 8
    rows = 777
    n = MANY // (width // lanes) + 5
    x = made(rows, width, dtype, width)
    g = torch.Generator(device="cuda").manual_seed(width)
    idx = torch.randint(0, rows, (n,), generator=g, device="cuda", dtype=torch.int32)
    idx[::101] = -1
    idx[50::101] = rows
    idx[n - 1] = rows - 1
    codes, scale = ops.quantize_rows(x, rows=idx)
    want, s = plain(x)
    ok = (idx >= 0) & (idx < rows)
    at = torch.where(ok, idx, 0).long()
    assert torch.equal(scale, torch.where(ok, s[at], torch.zeros_like(s[at])))
    assert torch.equal(codes, torch.where(ok[:, None], want[at], torch.zeros_like(want[at])))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("width", [1024, 1023])
def test_large_not_finite(ops, dtype, width):
    """NaN and infinities among many rows: their own scale and codes, and no one else's."""
    rows = 8200
    x = made(rows, width, dtype, 1)
    x[100, 17], x[4000, 0], x[rows - 1, width - 1] = float("nan"), float("inf"), float("-inf")
    codes, scale = ops.quantize_rows(x)
    want, s = plain(torch.nan_to_num(x, 0, 0, 0))
    assert torch.isnan(scale[100]) and scale[4000] == float("inf") and scale[rows - 1] == float("inf")
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[[100, 4000, rows - 1]] = False
    assert int(codes[~keep].abs().max()) == 0
    assert torch.equal(codes[keep], want[keep]) and torch.equal(scale[keep], s[keep])
