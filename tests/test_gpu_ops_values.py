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
