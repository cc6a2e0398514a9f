"""Token operators at values where an output can lose its last places: SwiGLU far from zero, scales near the smallest
normal number.  Every kernel that a product can take: few tokens, tiles alone and split over clusters, pairs of CTAs, layouts
that start at any byte."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ptq_int8_lab_b200.ops import Int8Ops
    return Int8Ops(0)


# rows, in_features, bytes between rows beyond them: what the comment says of B200's choice
PATHS = [pytest.param(1, 96, 0, id="few"), pytest.param(4, 512, 0, id="few4"), pytest.param(9, 4096, 0, id="split"),
         pytest.param(40, 64, 0, id="tile"), pytest.param(900, 256, 0, id="wide"), pytest.param(5, 97, 3, id="any")]


def strided(rows, cols, pad, dtype=torch.int8):
    return torch.zeros((rows, cols + pad), dtype=dtype, device="cuda")[:, :cols]


@pytest.mark.parametrize("rows,k,pad", PATHS)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("up", [1.0, -3.5, 1e30])
def test_swiglu_over_the_range(ops, rows, k, pad, bits, up):
    """silu(g) * u in 32 bits for gates from far below to far above zero, against 64 bits.

    All codes are zero, so gate and up are the bias itself.  Bounds in units of 2^-23.  Up to |g| = 64, g / (1 + e): the
    power of two 2 and its correction 1/2, the sum 1/2, the reciprocal 1, the products with g and u 1/2 each: 5.  Below,
    g exp(g): the exponential 2 and half a unit each for exp(-64) and three products: 4.  Steps that are subnormal there
    add half of 2^-149 each, scaled by u where u comes after them."""
    g = np.concatenate([np.linspace(-110, 100, 2101), -87.3 - np.arange(0, 5, 0.01), [0.0, -0.0, 1e-30, -1e-30, 3e38, -3e38,
                        -64.0, np.nextafter(np.float32(-64), np.float32(-65)), -88.72, -88.73, -1e5, 1e5]]).astype(np.float32)
    n = len(g)
    width = k if bits == 8 else (k + 1) // 2
    bias = torch.from_numpy(np.concatenate([g, np.full(n, up, np.float32)])).cuda()
    y = ops.linear(strided(rows, k, pad), torch.ones(rows, device="cuda"),
                   strided(2 * n, width, pad, torch.int8 if bits == 8 else torch.uint8), torch.ones(2 * n, device="cuda"),
                   bias=bias, bits=bits, act=1, dtype=torch.float32).cpu().numpy()
    g64, u = g.astype(np.float64), float(np.float32(up))
    with np.errstate(over="ignore"):
        want = g64 / (1 + np.exp(-g64)) * u
    inside = np.abs(want) < 3.4e38   # the others overflow to infinity, as the definition does
    tol = np.abs(want) * 5 * 2.0 ** -23 * (1 + 1e-6) + 2.0 ** -149 * (1 + abs(u))
    assert np.all(np.abs(y.astype(np.float64) - want)[:, inside] <= tol[inside])
    assert np.all(y[:, ~inside] == np.where(want[~inside] > 0, np.inf, -np.inf).astype(np.float32))


def pack4(c):
    """int8 codes in [-8, 7] -> two per byte, the even one in the low half."""
    if c.shape[-1] % 2:
        c = np.concatenate([c, np.zeros((*c.shape[:-1], 1), np.int8)], axis=-1)
    return ((c[..., 0::2] & 15) | ((c[..., 1::2] & 15) << 4)).astype(np.uint8)


@pytest.mark.parametrize("rows,k,pad", PATHS)
@pytest.mark.parametrize("bits", [8, 4])
def test_scales_near_the_smallest_normal_number(ops, rows, k, pad, bits):
    """Products of scales from 2^-150 to 2^-120, so normal, subnormal and zero ones: bit for bit the definition's two
    roundings in numpy's 32 bits, on every kernel."""
    rng = np.random.default_rng(rows + bits)
    n = 300
    x = rng.integers(-128, 128, (rows, k), dtype=np.int8)
    w = rng.integers(-8, 8, (n, k), dtype=np.int8)
    xs = np.exp2(rng.uniform(-65, -60, rows)).astype(np.float32)
    ws = np.exp2(rng.uniform(-85, -60, n)).astype(np.float32)
    xd, wc = strided(rows, k, pad), w if bits == 8 else pack4(w)
    xd.copy_(torch.from_numpy(x))
    wd = strided(*wc.shape, pad, torch.int8 if bits == 8 else torch.uint8)
    wd.copy_(torch.from_numpy(wc))
    y = ops.linear(xd, torch.from_numpy(xs).cuda(), wd, torch.from_numpy(ws).cuda(), bits=bits, dtype=torch.float32).cpu().numpy()
    acc = (x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float32)
    want = acc * (xs[:, None] * ws[None, :])
    assert np.array_equal(y.view(np.int32), (want + np.float32(0)).view(np.int32))
