"""Token operators (quantize_rows, linear, linear_grouped) against plain 64-bit implementations.

Codes, scales and products without SwiGLU have to be equal bit for bit: the sums are exact integers and each
further step of the definition is one IEEE rounding that numpy repeats.  SwiGLU is compared with its 64-bit value
on the same 32-bit gate and up values; its tolerance is the sum of the bounds of its steps (see swiglu_close).
"""
import numpy as np
import pytest
import torch

from ptq_int8_lab_b200 import engine as E

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    from ptq_int8_lab_b200.ops import Int8Ops
    return Int8Ops(0)


# ------------------------------------------------------------------ plain forms

def plain_rows(x):
    """(codes, scale) of float rows: the definition, the quotient in float64."""
    x = x.astype(np.float32)
    with np.errstate(all="ignore"):
        top = np.abs(x).max(axis=1)
        finite = np.isfinite(top)
        scale = np.maximum(top / np.float32(127), np.float32(1e-8))
        scale = np.where(finite, scale, np.where(np.isnan(x).any(axis=1), np.float32(np.nan), np.float32(np.inf)))
        q = x.astype(np.float64) / scale.astype(np.float64)[:, None]
        codes = np.where(q >= 0, np.floor(q + 0.5), np.ceil(q - 0.5))
        codes = np.where(finite[:, None], codes, 0)
    return codes.astype(np.int8), scale.astype(np.float32)


def plain_sums(x, w):
    """Exact: every partial sum is an integer below 2^53."""
    return (torch.from_numpy(x).double() @ torch.from_numpy(w).double().t()).numpy()


def plain_product(x, xs, w, ws, bias):
    acc = plain_sums(x, w).astype(np.float32)
    y = acc * (xs[:, None] * ws[None, :])
    return y if bias is None else y + bias[None, :]


def swiglu_close(got, z, n):
    """got (f32) against silu(g) * u in float64.  Steps and their bounds, in ulps of 2^-23: exp 2 + 1.16 |g|, the sum 1,
    the quotient 2, the product 1.  Below the smallest normal number (where the quotient may flush) the difference is
    absolute."""
    g, u = z[:, :n].astype(np.float64), z[:, n:].astype(np.float64)
    with np.errstate(over="ignore"):
        want = g / (1.0 + np.exp(-g)) * u
    tol = np.abs(want) * ((6 + 1.16 * np.abs(g)) * 2.0 ** -23) * (1 + 1e-6) + 1e-37 * (1 + np.abs(u))
    assert np.all(np.abs(got.astype(np.float64) - want) <= tol)


def to_type(y, dtype):
    return torch.from_numpy(y).to(DT[dtype])


def pack4(c):
    """int8 codes in [-8, 7] -> two per byte, the even one in the low half."""
    if c.shape[-1] % 2:
        c = np.concatenate([c, np.zeros((*c.shape[:-1], 1), np.int8)], axis=-1)
    return ((c[..., 0::2] & 15) | ((c[..., 1::2] & 15) << 4)).astype(np.uint8)


def laid(a, pitch=0, start=0):
    """A device copy whose last dimension has a pitch (0: rounded up to 16 elements) and whose data starts `start`
    elements into its buffer."""
    a = torch.from_numpy(np.ascontiguousarray(a))
    pitch = pitch or (a.shape[-1] + 15) // 16 * 16
    lead = a.shape[:-1]
    buf = torch.full((int(np.prod(lead)) * pitch + start + 16,), 85, dtype=a.dtype, device="cuda")
    t = buf[start:start + int(np.prod(lead)) * pitch].view(*lead, pitch)[..., :a.shape[-1]]
    t.copy_(a)
    return t


def case(rng, rows, k, n, bits, gated, bias, groups=0):
    lead = (groups,) if groups else ()
    ch = 2 * n if gated else n
    lo, hi = (-128, 128) if bits == 8 else (-8, 8)
    x = rng.integers(-128, 128, (rows, k), dtype=np.int8)
    w = rng.integers(lo, hi, (*lead, ch, k), dtype=np.int8)
    # products near 1, so that SwiGLU sees both sides of its curve
    xs = rng.uniform(0.2, 2.0, rows).astype(np.float32)
    ws = (rng.uniform(0.2, 2.0, (*lead, ch)) / (70 * (70 if bits == 8 else 4.6) * np.sqrt(k))).astype(np.float32)
    b = rng.normal(0, 1, (*lead, ch)).astype(np.float32) if bias else None
    return x, xs, w, ws, b


def dev(a):
    return None if a is None else torch.from_numpy(a).cuda()


def same(got, want):
    bits = {4: torch.int32, 2: torch.int16}[want.element_size()]
    assert got.dtype == want.dtype and torch.equal(got.contiguous().view(bits), want.contiguous().view(bits)), \
        (got.float() - want.float()).abs().max()


def check(call, z, n, gated, dtype):
    """call(dtype) -> y.  With SwiGLU: the 32-bit output against 64 bits, the 16-bit ones equal to it rounded once."""
    got = call(DT[dtype]).cpu()
    if not gated:
        same(got, to_type(z, dtype))
        return
    whole = got if dtype == "f32" else call(torch.float32).cpu()
    swiglu_close(whole.numpy(), z, n)
    same(got, whole.to(DT[dtype]))


# ------------------------------------------------------------------ quantize_rows

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("width", [1, 2, 7, 8, 15, 16, 31, 64, 100, 127, 128, 129, 255, 256, 1001, 1024, 2047, 4096, 8200, 16385,
                                   40000])
def test_rows_widths(ops, dtype, width):
    rng = np.random.default_rng(width)
    x = torch.from_numpy(rng.normal(0, 1, (5, width)).astype(np.float32)).to(DT[dtype])
    x[2] *= 37
    codes, scale = ops.quantize_rows(x.cuda())
    want, ws = plain_rows(x.float().numpy())
    assert np.array_equal(scale.cpu().numpy(), ws)
    assert np.array_equal(codes.cpu().numpy(), want)
    assert codes.stride(0) % 16 == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("width,pitch,start,cpitch,cstart", [(64, 64, 0, 64, 0), (64, 72, 0, 80, 0), (64, 65, 0, 64, 0),
                                                             (64, 64, 1, 64, 0), (64, 64, 0, 67, 0), (64, 64, 0, 64, 3),
                                                             (333, 333, 5, 333, 7), (4100, 4103, 3, 4112, 0),
                                                             (513, 520, 8, 513, 8), (2048, 2049, 1, 2049, 1)])
def test_rows_layouts(ops, dtype, width, pitch, start, cpitch, cstart):
    rng = np.random.default_rng(width + pitch)
    x = torch.from_numpy(rng.normal(0, 2, (9, width)).astype(np.float32)).to(DT[dtype])
    buf = torch.full((9 * pitch + start,), 1e4, dtype=DT[dtype], device="cuda")
    xd = buf[start:start + 9 * pitch].view(9, pitch)[:, :width]
    xd.copy_(x)
    cbuf = torch.full((9 * cpitch + cstart,), 77, dtype=torch.int8, device="cuda")
    codes = cbuf[cstart:].view(9, cpitch)[:, :width]
    scale = torch.empty(9, device="cuda")
    ops.quantize_rows(xd, out=(codes, scale))
    want, ws = plain_rows(x.float().numpy())
    assert np.array_equal(codes.cpu().numpy(), want)
    assert np.array_equal(scale.cpu().numpy(), ws)
    whole = cbuf.cpu().numpy()
    assert np.all(whole[:cstart] == 77) and np.all(whole[cstart:].reshape(9, cpitch)[:, width:] == 77)


@pytest.mark.parametrize("width", [96, 97, 2048])
def test_rows_gather(ops, width):
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.normal(0, 1, (11, width)).astype(np.float32)).to(torch.bfloat16)
    idx = np.array([3, 3, 0, 10, -1, 11, 7, 2 ** 31 - 1, -2 ** 31, 5, 5, 5, 1], np.int32)
    codes, scale = ops.quantize_rows(x.cuda(), rows=torch.from_numpy(idx).cuda())
    want, ws = plain_rows(x.float().numpy())
    ok = (idx >= 0) & (idx < 11)
    i = np.where(ok, idx, 0)
    assert np.array_equal(codes.cpu().numpy(), np.where(ok[:, None], want[i], 0))
    assert np.array_equal(scale.cpu().numpy(), np.where(ok, ws[i], 0))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("width", [40, 257, 4096])
def test_rows_extremes(ops, dtype, width):
    """Zero rows, denormals, the type's largest value, NaN and infinities of both signs."""
    big = float(torch.finfo(DT[dtype]).max)
    x = torch.zeros((9, width))
    x[1] = torch.linspace(-1e-9, 1e-9, width)
    x[2, ::3], x[2, 1::3] = big, -big
    x[3] = 1.0
    x[3, width // 2] = float("nan")
    x[4] = -1.0
    x[4, 0] = float("inf")
    x[5, width - 1] = float("-inf")
    x[6, 0], x[6, width - 1] = float("inf"), float("nan")
    x[7] = torch.arange(width) % 128
    x[8] = -x[7] - 0.5
    x = x.to(DT[dtype])
    codes, scale = ops.quantize_rows(x.cuda())
    want, ws = plain_rows(x.float().numpy())
    assert np.array_equal(codes.cpu().numpy(), want)
    assert np.array_equal(scale.cpu().numpy(), ws, equal_nan=True)
    assert np.isnan(ws[3]) and np.isinf(ws[4]) and np.isinf(ws[5]) and np.isnan(ws[6])


def test_rows_ties(ops):
    """Every neighbour of every rounding boundary, at scales of all kinds of mantissa."""
    rng = np.random.default_rng(3)
    tops = np.concatenate([np.float32(127) * np.float32(2.0) ** np.arange(-6, 6), rng.uniform(0.01, 900, 60)]).astype(np.float32)
    rows = []
    for t in tops:
        s = np.maximum(t / np.float32(127), np.float32(1e-8))
        b = ((np.arange(-127, 127) + 0.5) * np.float64(s)).astype(np.float32)
        near = [b] + [np.nextafter(b, np.float32(d)) for d in (-np.inf, np.inf)]
        row = np.concatenate([*near, [t]])
        rows.append(np.clip(row, -t, t))
    x = np.stack(rows).astype(np.float32)
    codes, scale = ops.quantize_rows(dev(x))
    want, ws = plain_rows(x)
    assert np.array_equal(scale.cpu().numpy(), ws)
    assert np.array_equal(codes.cpu().numpy(), want)


def test_rows_none(ops):
    codes, scale = ops.quantize_rows(torch.empty((0, 64), device="cuda"))
    assert codes.shape == (0, 64) and scale.shape == (0,)
    codes, scale = ops.quantize_rows(torch.ones((3, 64), device="cuda"), rows=torch.empty(0, dtype=torch.int32, device="cuda"))
    assert codes.shape == (0, 64)


# ------------------------------------------------------------------ linear

SHAPES = [(1, 1, 1), (1, 64, 5), (1, 4096, 130), (2, 129, 128), (3, 31, 257), (4, 512, 384), (5, 1000, 129), (7, 2048, 64),
          (8, 272, 300), (9, 640, 131), (16, 128, 256), (17, 130, 100), (31, 1024, 512), (33, 96, 127), (64, 2000, 640),
          (65, 513, 513), (100, 256, 128), (128, 384, 512), (129, 160, 257), (200, 4096, 96), (256, 1040, 520),
          (257, 127, 255), (300, 2064, 1030), (520, 640, 777), (1025, 144, 300)]


@pytest.mark.parametrize("rows,k,n", SHAPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("gated", [False, True])
def test_linear_shapes(ops, rows, k, n, bits, gated):
    rng = np.random.default_rng(rows * 7 + k * 3 + n)
    dtype = ["bf16", "f16", "f32"][(rows + n) % 3]
    bias = bool(k % 3)
    x, xs, w, ws, b = case(rng, rows, k, n, bits, gated, bias)
    wd = laid(w if bits == 8 else pack4(w))
    a = (laid(x), dev(xs), wd, dev(ws), dev(b))
    check(lambda t: ops.linear(*a, bits=bits, act=1 if gated else 0, dtype=t), plain_product(x, xs, w, ws, b), n, gated, dtype)


@pytest.mark.parametrize("rows,k,n", [(2500, 272, 2100), (5000, 130, 1111), (4097, 640, 1290), (9000, 48, 530),
                                      (700, 8192, 500), (130, 16384, 260), (48, 8200, 1000), (300, 300, 5000),
                                      (20, 4096, 9000), (1000, 2000, 130)])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("gated", [False, True])
def test_linear_many_tiles(ops, rows, k, n, bits, gated):
    """More tiles than the device runs at once, so that every CTA takes several; and few tiles with long sums, which
    clusters share."""
    rng = np.random.default_rng(rows)
    x, xs, w, ws, b = case(rng, rows, k, n, bits, gated, True)
    a = (laid(x), dev(xs), laid(w if bits == 8 else pack4(w)), dev(ws), dev(b))
    check(lambda t: ops.linear(*a, bits=bits, act=1 if gated else 0, dtype=t), plain_product(x, xs, w, ws, b), n, gated, "bf16")


@pytest.mark.parametrize("counts", [[900, 0, 3, 2000, 1, 515, 30, 1300], [257] * 20], ids=["uneven", "even"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("gated", [False, True])
def test_grouped_many_tiles(ops, counts, bits, gated):
    rng = np.random.default_rng(len(counts))
    offs = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    k, n = 400, 1000
    x, xs, w, ws, b = case(rng, int(offs[-1]), k, n, bits, gated, True, len(counts))
    a = (laid(x), dev(xs), dev(offs), laid(w if bits == 8 else pack4(w)), dev(ws), dev(b))
    check(lambda t: ops.linear_grouped(*a, bits=bits, act=1 if gated else 0, dtype=t), plain_grouped(x, xs, offs, w, ws, b), n,
          gated, "f16")


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows", [1, 6, 40, 300])
@pytest.mark.parametrize("layout", ["odd pitches", "odd starts", "wide pitches"])
def test_linear_layouts(ops, bits, gated, rows, layout):
    rng = np.random.default_rng(rows)
    k, n = 331, 190
    x, xs, w, ws, b = case(rng, rows, k, n, bits, gated, True)
    wc = w if bits == 8 else pack4(w)
    px, pw, s = {"odd pitches": (k, wc.shape[-1] + 1, 0), "odd starts": (0, 0, 5), "wide pitches": (1024, 512, 16)}[layout]
    a = (laid(x, px, s), dev(xs), laid(wc, pw, s), dev(ws), dev(b))

    def call(t):
        ybuf = torch.full((rows, n + 9), 7.0, dtype=t, device="cuda")
        y = ops.linear(*a, bits=bits, act=1 if gated else 0, out=ybuf[:, 3:3 + n])
        rest = ybuf.cpu()
        assert torch.all(rest[:, :3] == 7) and torch.all(rest[:, 3 + n:] == 7)
        return y

    check(call, plain_product(x, xs, w, ws, b), n, gated, "bf16")


@pytest.mark.parametrize("rows", [1, 5, 130])
@pytest.mark.parametrize("bits", [8, 4])
def test_linear_largest_sums(ops, rows, bits):
    """The longest row that is accepted, all codes at -128 (-8): the sum is the largest that there is."""
    k, low = 131071, -128 if bits == 8 else -8
    x = np.full((rows, k), -128, np.int8)
    w = np.full((3, k), low, np.int8)
    w[1] = -low - 1
    one = np.ones(3, np.float32)
    y = ops.linear(laid(x), torch.ones(rows, device="cuda"), laid(w if bits == 8 else pack4(w)), dev(one), bits=bits,
                   dtype=torch.float32)
    want = np.float32([-128 * low * k, -128 * (-low - 1) * k, -128 * low * k])
    assert np.array_equal(y.cpu().numpy(), np.tile(want, (rows, 1)))


def test_linear_rejects_longer_sums(ops):
    k = 131072
    with pytest.raises(E.Ptq8Error, match="in_features"):
        ops.linear(torch.zeros((1, k), dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"),
                   torch.zeros((1, k), dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))


@pytest.mark.parametrize("rows", [2, 140])
def test_linear_not_finite_rows(ops, rows):
    """A token with scale NaN or infinity gives NaN in its own row only; one with scale 0 gives the bias."""
    rng = np.random.default_rng(0)
    x, xs, w, ws, b = case(rng, rows, 256, 200, 8, False, True)
    clean = plain_product(x, xs, w, ws, b)
    x[0], xs[0] = 0, np.inf
    y = ops.linear(laid(x), dev(xs), laid(w), dev(ws), bias=dev(b), dtype=torch.float32).cpu().numpy()
    assert np.isnan(y[0]).all() and np.array_equal(y[1:], clean[1:])
    xs[0], xs[1] = np.nan, 0
    y = ops.linear(laid(x), dev(xs), laid(w), dev(ws), bias=dev(b), dtype=torch.float32).cpu().numpy()
    assert np.isnan(y[0]).all() and np.array_equal(y[1], b) and np.array_equal(y[2:], clean[2:])


@pytest.mark.parametrize("rows", [4, 200])
def test_swiglu_saturates(ops, rows):
    """Gates far below and above zero: silu goes to -0 and to the gate itself, without NaN."""
    k, n = 64, 130
    x = np.full((rows, k), 127, np.int8)
    w = np.ones((2 * n, k), np.int8)
    w[1:n:2] = -1
    ws = np.full(2 * n, 1.0, np.float32)
    xs = np.linspace(0.001, 4, rows).astype(np.float32)
    y = ops.linear(laid(x), dev(xs), laid(w), dev(ws), act=1, dtype=torch.float32)
    z = plain_product(x, xs, w, ws, None)
    assert torch.isfinite(y).all()
    swiglu_close(y.cpu().numpy(), z, n)


def test_linear_far_rows(ops):
    """Row offsets past 2^31 elements in x and y."""
    rows, k, n, pitch = 70001, 48, 24, 32768
    xb = torch.zeros((rows, pitch), dtype=torch.int8, device="cuda")
    yb = torch.zeros((rows, pitch), dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(1)
    x, xs, w, ws, _ = case(rng, rows, k, n, 8, False, False)
    xb[:, 128:128 + k] = dev(x)
    y = ops.linear(xb[:, 128:128 + k], dev(xs), laid(w), dev(ws), out=yb[:, 1:1 + n])
    same(y.cpu(), to_type(plain_product(x, xs, w, ws, None), "bf16"))
    assert int(torch.count_nonzero(yb[-1, 1 + n:])) == 0
    codes, scale = ops.quantize_rows(yb[:, 1:1 + n], out=(xb[:, :n], torch.empty(rows, device="cuda")))
    want, s = plain_rows(y.float().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), want) and np.array_equal(scale.cpu().numpy(), s)


def test_linear_none(ops):
    y = ops.linear(torch.empty((0, 64), dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda"),
                   torch.zeros((32, 64), dtype=torch.int8, device="cuda"), torch.ones(32, device="cuda"))
    assert y.shape == (0, 32)


# ------------------------------------------------------------------ linear_grouped

def plain_grouped(x, xs, offs, w, ws, b):
    z = np.zeros((x.shape[0], w.shape[1]), np.float32)
    for g in range(w.shape[0]):
        a, e = offs[g], offs[g + 1]
        z[a:e] = plain_product(x[a:e], xs[a:e], w[g], ws[g], None if b is None else b[g])
    return z


COUNTS = [[1], [0, 3], [0, 0, 0, 5, 0], [1, 1, 1, 1, 1, 1, 1, 1], [16, 0, 17, 1, 64], [130, 2, 0, 257, 31], [300],
          [0, 700, 1], [3] * 40, [0] * 63 + [9], [128, 128, 128, 128], [33, 129, 513, 5]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("k,n", [(96, 130), (520, 257), (1024, 128)])
def test_grouped(ops, counts, bits, gated, k, n):
    rng = np.random.default_rng(sum(counts) + k)
    offs = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    rows = int(offs[-1])
    dtype = ["bf16", "f16", "f32"][(rows + n) % 3]
    x, xs, w, ws, b = case(rng, rows, k, n, bits, gated, len(counts) % 2 == 0, len(counts))
    a = (laid(x), dev(xs), dev(offs), laid(w if bits == 8 else pack4(w)), dev(ws), dev(b))
    check(lambda t: ops.linear_grouped(*a, bits=bits, act=1 if gated else 0, dtype=t), plain_grouped(x, xs, offs, w, ws, b), n,
          gated, dtype)


@pytest.mark.parametrize("pitch", [0, 203])
@pytest.mark.parametrize("offs", [[5, 5, 20, 31], [0, 0, 0, 0], [-9, 4, 10, 1000], [40, 41, 42, 43]])
def test_grouped_uncovered_rows(ops, offs, pitch):
    """Rows of no group keep what they held; offsets outside [0, rows] are clamped."""
    rng = np.random.default_rng(2)
    rows, k, n = 40, 200, 70
    x, xs, w, ws, _ = case(rng, rows, k, n, 8, False, False, 3)
    y = torch.full((rows, n), 9.0, device="cuda")
    ops.linear_grouped(laid(x, pitch), dev(xs), torch.tensor(offs, dtype=torch.int32, device="cuda"), laid(w, pitch), dev(ws), out=y)
    clamped = np.clip(offs, 0, rows)
    want = plain_grouped(x, xs, clamped, w, ws, None)
    inside = (np.arange(rows) >= clamped[0]) & (np.arange(rows) < clamped[-1])
    want[~inside] = 9.0
    assert np.array_equal(y.cpu().numpy(), want)


@pytest.mark.parametrize("pitch", [0, 131])
def test_grouped_strided_groups(ops, pitch):
    """Groups further apart than their weights; offsets that decrease leave empty groups and stay in bounds."""
    rng = np.random.default_rng(4)
    x, xs, w, ws, _ = case(rng, 24, 128, 65, 8, False, False, 4)
    big = laid(np.concatenate([w, np.full((4, 7, 128), 99, np.int8)], axis=1), pitch)[:, :65]
    offs = np.array([0, 10, 4, 4, 24], np.int32)
    y = ops.linear_grouped(laid(x), dev(xs), dev(offs), big, dev(ws), dtype=torch.float32).cpu().numpy()
    # rows 4..9 belong to groups 0 and 3: either may be the last to write them
    for a, e, g in ((0, 4, 0), (10, 24, 3)):
        assert np.array_equal(y[a:e], plain_product(x[a:e], xs[a:e], w[g], ws[g], None))


# ------------------------------------------------------------------ streams, graphs, refusals

def test_streams_and_order(ops):
    """quantize -> product chains on two streams at once, each in its own order."""
    rng = np.random.default_rng(8)
    k, n = 1024, 512
    _, _, w, ws, _ = case(rng, 1, k, n, 8, False, False)
    wd, wsd = laid(w), dev(ws)
    xs_in = [torch.from_numpy(rng.normal(0, 1, (r, k)).astype(np.float32)).cuda() for r in (3, 250)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs_in]
    outs = []
    for s, x in zip(streams, xs_in):
        with torch.cuda.stream(s):
            for _ in range(10):
                codes, scale = ops.quantize_rows(x)
                y = ops.linear(codes, scale, wd, wsd, dtype=torch.float32)
            outs.append(y)
    torch.cuda.synchronize()
    for x, y in zip(xs_in, outs):
        c, s = plain_rows(x.cpu().numpy())
        assert np.array_equal(y.cpu().numpy(), plain_product(c, s, w, ws, None))
    y = torch.empty((3, n), device="cuda")
    codes, scale = ops.quantize_rows(xs_in[0])
    torch.cuda.synchronize()
    ops.linear(codes, scale, wd, wsd, out=y, stream=streams[0])
    ops.check_device_error(streams[0])
    assert torch.equal(y, outs[0])
    with pytest.raises(E.Ptq8Error, match="out is wanted"):
        ops.linear(codes, scale, wd, wsd, stream=streams[0])


def test_weights_made_by_the_call_before(ops):
    """Weights quantized on the device by the launch just before the product that reads them."""
    rng = np.random.default_rng(12)
    for rows in (2, 256):
        x, xs, _, _, _ = case(rng, rows, 2048, 1, 8, False, False)
        xd, xsd = laid(x), dev(xs)
        for i in range(4):
            wf = rng.normal(0, 1 + i, (640, 2048)).astype(np.float32)
            wfd = dev(wf)
            w, ws = ops.quantize_rows(wfd)
            y = ops.linear(xd, xsd, w, ws, dtype=torch.float32)
            c, s = plain_rows(wf)
            assert np.array_equal(y.cpu().numpy(), plain_product(x, xs, c, s, None))


def test_graph(ops):
    """The whole chain captured once and replayed on new inputs."""
    rng = np.random.default_rng(9)
    rows, k, n = 40, 512, 384
    _, _, w, ws, _ = case(rng, 1, k, n, 8, True, False)
    w2 = rng.integers(-128, 128, (k, n), dtype=np.int8)
    ws2 = rng.uniform(1e-4, 1e-3, k).astype(np.float32)
    wd, wsd, w2d, ws2d = laid(w), dev(ws), laid(w2), dev(ws2)
    x = torch.zeros((rows, k), device="cuda")

    def chain():
        c, s = ops.quantize_rows(x)
        h = ops.linear(c, s, wd, wsd, act=1, dtype=torch.float32)
        c, s = ops.quantize_rows(h)
        return h, ops.linear(c, s, w2d, ws2d, dtype=torch.float32)

    chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, y = chain()
    for seed in range(3):
        xn = np.random.default_rng(seed).normal(0, 1, (rows, k)).astype(np.float32)
        x.copy_(torch.from_numpy(xn))
        graph.replay()
        torch.cuda.synchronize()
        c, s = plain_rows(xn)
        swiglu_close(h.cpu().numpy(), plain_product(c, s, w, ws, None), n)
        c, s = plain_rows(h.cpu().numpy())
        assert np.array_equal(y.cpu().numpy(), plain_product(c, s, w2, ws2, None))
    del graph


def test_same_outputs_every_time(ops):
    rng = np.random.default_rng(10)
    for rows, k, n, gated in ((3, 4096, 1024, False), (20, 4096, 512, True), (500, 1024, 700, True)):
        x, xs, w, ws, b = case(rng, rows, k, n, 8, gated, True)
        a = (laid(x), dev(xs), laid(w), dev(ws))
        first = ops.linear(*a, bias=dev(b), act=int(gated))
        for _ in range(5):
            assert torch.equal(first, ops.linear(*a, bias=dev(b), act=int(gated)))


@pytest.mark.parametrize("rows,k,n,gated", [(3000, 8192, 80, False), (2000, 4096, 600, False), (500, 4096, 512, True),
                                            (48, 8192, 1024, False)])
def test_int4_many_launches(ops, rows, k, n, gated):
    """int4 tiles whose loads come from cold memory, over and over: the stages that the unpacking warps share in turns
    hold each launch's own weights.  Four weight sets in turn, each output equal to its first."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    ch = 2 * n if gated else n
    x = torch.randint(-128, 128, (rows, k), generator=g, device="cuda", dtype=torch.int8)
    xs, ws = torch.rand(rows, generator=g, device="cuda") + 0.1, torch.rand(ch, generator=g, device="cuda") * 1e-5
    w = [torch.randint(0, 256, (ch, k // 2), generator=g, device="cuda", dtype=torch.uint8) for _ in range(4)]
    first = [ops.linear(x, xs, v, ws, bits=4, act=int(gated)) for v in w]
    flush = torch.empty(160 << 20, dtype=torch.uint8, device="cuda")
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(160):
        flush.fill_(i & 1)
        wrong += (ops.linear(x, xs, w[i % 4], ws, bits=4, act=int(gated)) != first[i % 4]).sum()
    assert int(wrong) == 0
    ops.check_device_error()


def _ok():
    z = lambda *s, t=torch.int8: torch.zeros(s, dtype=t, device="cuda")   # noqa: E731
    return dict(x=z(4, 64), x_scale=z(4, t=torch.float32), w=z(32, 64), w_scale=z(32, t=torch.float32))


@pytest.mark.parametrize("change,needle", [
    (dict(x=lambda a: a["x"].cpu()), "not on cuda:0"),
    (dict(x=lambda a: a["x"].float()), "dtype"),
    (dict(x=lambda a: a["x"][0]), "two dimensions"),
    (dict(x=lambda a: a["x"].t().contiguous().t()), "not consecutive"),
    (dict(x_scale=lambda a: a["x_scale"][:3]), "x_scale"),
    (dict(x_scale=lambda a: a["x_scale"].half()), "x_scale"),
    (dict(x_scale=lambda a: torch.zeros(8, device="cuda")[::2]), "not contiguous"),
    (dict(w=lambda a: a["w"][:, :63]), "63 bytes for 64"),
    (dict(w=lambda a: a["w"].to(torch.uint8)), "dtype"),
    (dict(w_scale=lambda a: a["w_scale"][:31]), "w_scale"),
    (dict(bits=lambda a: 2), "bits 2"),
    (dict(bits=lambda a: 4), "64 bytes for 64"),
    (dict(act=lambda a: 5), "act 5"),
    (dict(act=lambda a: 1, w=lambda a: a["w"][:31], w_scale=lambda a: a["w_scale"][:31]), "gate and up"),
    (dict(bias=lambda a: a["w_scale"][:30]), "bias"),
    (dict(dtype=lambda a: torch.float64), "dtype"),
    (dict(out=lambda a: torch.zeros((4, 31), device="cuda")), "out"),
    (dict(out=lambda a: torch.zeros((4, 32), device="cuda", dtype=torch.float64)), "out"),
])
def test_linear_refusals(ops, change, needle):
    a = _ok()
    new = {k: f(a) for k, f in change.items()}
    with pytest.raises(E.Ptq8Error, match=needle):
        ops.linear(**{**a, **new})


@pytest.mark.parametrize("change,needle", [
    (dict(offsets=lambda a: None), "offsets"),
    (dict(offsets=lambda a: a["offsets"].long()), "offsets"),
    (dict(offsets=lambda a: a["offsets"][:2]), "offsets"),
    (dict(offsets=lambda a: a["offsets"].cpu()), "offsets"),
    (dict(w=lambda a: a["w"][0]), "groups, channels, in"),
    (dict(w=lambda a: a["w"][:1].expand(2, 32, 64)), "groups overlap"),
    (dict(w_scale=lambda a: a["w_scale"][0]), "w_scale"),
])
def test_grouped_refusals(ops, change, needle):
    a = _ok()
    a["w"], a["w_scale"] = torch.stack([a["w"]] * 2), torch.stack([a["w_scale"]] * 2)
    a["offsets"] = torch.tensor([0, 1, 4], dtype=torch.int32, device="cuda")
    new = {k: f(a) for k, f in change.items()}
    with pytest.raises(E.Ptq8Error, match=needle):
        ops.linear_grouped(**{**a, **new})


def test_too_many_groups(ops):
    a = _ok()
    w = torch.zeros((1025, 1, 64), dtype=torch.int8, device="cuda")
    with pytest.raises(E.Ptq8Error, match="groups 1025"):
        ops.linear_grouped(a["x"], a["x_scale"], torch.zeros(1026, dtype=torch.int32, device="cuda"), w,
                           torch.zeros((1025, 1), device="cuda"))


@pytest.mark.parametrize("args,needle", [
    (lambda x: dict(x=x.cpu()), "not on cuda:0"),
    (lambda x: dict(x=x.double()), "dtype"),
    (lambda x: dict(x=x[0]), "two dimensions"),
    (lambda x: dict(x=x.t()), "not consecutive"),
    (lambda x: dict(x=x, rows=torch.zeros(3, dtype=torch.int64, device="cuda")), "rows"),
    (lambda x: dict(x=x, out=(torch.zeros((4, 63), dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda"))), "codes"),
    (lambda x: dict(x=x, out=(torch.zeros((4, 64), dtype=torch.uint8, device="cuda"), torch.zeros(4, device="cuda"))), "codes"),
    (lambda x: dict(x=x, out=(torch.zeros((4, 64), dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda"))), "scale"),
    (lambda x: dict(x=x[:, :0]), "width 0"),
])
def test_rows_refusals(ops, args, needle):
    with pytest.raises(E.Ptq8Error, match=needle):
        ops.quantize_rows(**args(torch.zeros((4, 64), device="cuda")))


def test_handles(ops):
    from ptq_int8_lab_b200.ops import Int8Ops
    with pytest.raises(E.Ptq8Error):
        Int8Ops(4096)
    assert torch.zeros(1, device="cuda").item() == 0   # the refusal left no error behind
    L = E.lib()
    assert L.ptq8_linear(None, None, None) == 1 and L.ptq8_quantize_rows(None, None, None) == 1
    assert L.ptq8_linear(ops._h, None, None) == 1 and L.ptq8_linear_grouped(ops._h, None, None) == 1
    assert L.ptq8_quantize_rows(ops._h, None, None) == 1


@pytest.mark.parametrize("rows", [1, 2, 3, 4])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("k,n,pitch", [(2001, 130, 2016), (1023, 33, 1024), (511, 3, 512), (4112, 66, 4112), (1024, 1, 1024),
                                       (17, 7, 32), (2016, 130, 2016), (4096, 50, 8192)])
def test_few_tokens_row_ends(ops, rows, bits, gated, k, n, pitch):
    """Weights and codes whose last row ends with its buffer, and rows followed by bytes that must not count."""
    rng = np.random.default_rng(k + rows)
    x, xs, w, ws, b = case(rng, rows, k, n, bits, gated, True)

    def exact_end(a, p):
        """A device copy with pitch p whose buffer ends where its last row does."""
        a = torch.from_numpy(np.ascontiguousarray(a))
        buf = torch.full(((a.shape[0] - 1) * p + a.shape[1],), 85, dtype=a.dtype, device="cuda")
        t = buf.as_strided(a.shape, (p, 1))
        t.copy_(a)
        return t

    wc = w if bits == 8 else pack4(w)
    a = (exact_end(x, pitch), dev(xs), exact_end(wc, pitch if bits == 8 else (pitch // 2 + 15) // 16 * 16), dev(ws), dev(b))
    check(lambda t: ops.linear(*a, bits=bits, act=1 if gated else 0, dtype=t), plain_product(x, xs, w, ws, b), n, gated, "bf16")
