"""int4 products whose tiles two CTAs share, or whose unpacking warps take turns at the stages: launch after launch from
cold memory, each output equal to the exact product's."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ptq_int8_lab_b200.ops import Int8Ops
    return Int8Ops(0)


def widened(w):
    """[..., bytes] of packed codes -> [..., 2 * bytes] float64."""
    c = torch.stack((w & 15, w >> 4), dim=-1).flatten(-2).to(torch.int8)
    return torch.where(c > 7, c - 16, c).double()


def exact(x, xs, offs, w, ws):
    """The product before the epilogue, as 32-bit values: sums of integers, then the definition's two roundings."""
    y = torch.empty((x.shape[0], w.shape[1]), device="cuda")
    for g in range(w.shape[0]):
        a, b = offs[g], offs[g + 1]
        acc = (x[a:b].double() @ widened(w[g]).t()).float()
        y[a:b] = acc * (xs[a:b, None] * ws[g][None, :])
    return y


@pytest.mark.parametrize("counts,k,n,gated", [
    pytest.param([4096], 2048, 4096, False, id="pair of 256"), pytest.param([4096], 1024, 4096, True, id="pair of 128, gated"),
    pytest.param([3000], 640, 4200, True, id="pair of 128, gated, ragged"), pytest.param([2000], 4096, 600, False, id="tile of 128"),
    pytest.param([700, 0, 1000, 513, 1300], 1408, 2050, False, id="groups"),
    pytest.param([1200, 3, 0, 900, 1027], 1024, 2048, True, id="groups, gated")])
def test_int4_from_cold_memory(ops, counts, k, n, gated):
    """SwiGLU: near 1 its 32-bit steps stay within 8 units of 2^-23 of the value (5 for silu and the product, the rest for
    this form's own); four products of equal operands have to be equal bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(k + n)
    rows, groups, ch = sum(counts), len(counts), 2 * n if gated else n
    offs = [sum(counts[:i]) for i in range(groups + 1)]
    x = torch.randint(-128, 128, (rows, k), generator=g, device="cuda", dtype=torch.int8)
    xs = torch.rand(rows, generator=g, device="cuda") + 0.1
    ws = (torch.rand((groups, ch), generator=g, device="cuda") + 0.1) / (70 * 4.6 * k ** 0.5)
    sets = [torch.randint(0, 256, (groups, ch, k // 2), generator=g, device="cuda", dtype=torch.uint8) for _ in range(3)]
    od = torch.tensor(offs, dtype=torch.int32, device="cuda")

    def call(w):
        if groups == 1:
            return ops.linear(x, xs, w[0], ws[0], bits=4, act=int(gated), dtype=torch.float32)
        return ops.linear_grouped(x, xs, od, w, ws, bits=4, act=int(gated), dtype=torch.float32)

    want = []
    for w in sets:
        z = exact(x, xs, offs, w, ws)
        if gated:
            gate, up = z.double().chunk(2, dim=1)
            z = gate / (1 + torch.exp(-gate)) * up
            got = call(w)
            assert torch.all((got.double() - z).abs() <= z.abs() * 8 * 2.0 ** -23 + 1e-37)
            z = got
        want.append(z)
    flush = torch.empty(160 << 20, dtype=torch.uint8, device="cuda")
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(300):
        if i % 2:
            flush.fill_(i & 255)
        wrong += (call(sets[i % 3]) != want[i % 3]).sum()
    assert int(wrong) == 0
    ops.check_device_error()


@pytest.mark.parametrize("rows,k,n,act", [(4096, 512, 4096, 1), (4096, 2048, 4096, 0)])
def test_wait_runs_out(ops, rows, k, n, act):
    """A pair whose first load never comes gives up in both CTAs, and the next call is right again."""
    from ptq_int8_lab_b200 import engine as E
    g = torch.Generator(device="cuda").manual_seed(1)
    ch = 2 * n if act else n
    x = torch.randint(-128, 128, (rows, k), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(0, 256, (ch, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    xs, ws = torch.ones(rows, device="cuda"), torch.full((ch,), 1e-5, device="cuda")
    good = ops.linear(x, xs, w, ws, bits=4, act=act)
    ops.check_device_error()
    ops.set_wait_test(10_000_000, True)
    ops.linear(x, xs, w, ws, bits=4, act=act)
    with pytest.raises(E.Ptq8Error, match="ran out"):
        ops.check_device_error()
    ops.set_wait_test()
    assert torch.equal(ops.linear(x, xs, w, ws, bits=4, act=act), good)
    ops.check_device_error()
