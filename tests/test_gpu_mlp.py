"""The quantized MLPs: their layers put together by hand from the operators' definitions, in 64 bits."""
import numpy as np
import pytest
import torch

from ptq_int8_lab_b200 import engine as E

pytestmark = pytest.mark.gpu


def _weights(rng, experts, hidden, width):
    w1 = (rng.normal(0, 1, (experts, 2 * width, hidden)) / np.sqrt(hidden)).astype(np.float32)
    w2 = (rng.normal(0, 1, (experts, hidden, width)) / np.sqrt(width)).astype(np.float32)
    return w1, w2


def _codes(x):
    top = x.abs().amax(1, keepdim=True)
    s = (top / torch.full_like(top, 127.0)).clamp_min(1e-8)
    q = x.double() / s.double()
    return q.sign() * (q.abs() + 0.5).floor(), s.double()


def _plain(x, w1, w2, bits):
    """float64 MLP on the quantized weights and activations; the hidden state is kept in x's type."""
    def product(codes, scale, w):
        c, s = E.quantize_weight(w, bits)
        return (codes @ torch.from_numpy(c).double().t()) * scale * torch.from_numpy(s).double()
    z = product(*_codes(x.float()), w1)
    g, u = z.chunk(2, dim=1)
    h = (g / (1 + torch.exp(-g)) * u).to(x.dtype)
    return product(*_codes(h.float()), w2)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens", [1, 5, 130])
def test_dense(bits, tokens):
    """One code of the hidden state may differ by a step where a 32-bit hidden value differs in its last places: a
    step is 1/127 of its row's largest, so a row of `width` values moves by less than 1e-2 of its norm for any few."""
    from ptq_int8_lab_b200.mlp import Int8MLP
    rng = np.random.default_rng(tokens)
    w1, w2 = _weights(rng, 1, 320, 400)
    x = torch.from_numpy(rng.normal(0, 1, (tokens, 320)).astype(np.float32))
    got = Int8MLP(w1[0], w2[0], bits)(x.cuda()).cpu().double()
    want = _plain(x, w1[0], w2[0], bits)
    assert torch.linalg.norm(got - want) <= 1e-2 * torch.linalg.norm(want)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens,experts,top", [(1, 4, 2), (9, 8, 2), (64, 5, 3), (3, 16, 1)])
def test_experts(bits, tokens, experts, top):
    from ptq_int8_lab_b200.mlp import Int8Experts
    rng = np.random.default_rng(experts)
    w1, w2 = _weights(rng, experts, 256, 272)
    router = (rng.normal(0, 1, (experts, 256)) / 16).astype(np.float32)
    x = torch.from_numpy(rng.normal(0, 1, (tokens, 256)).astype(np.float32))
    layer = Int8Experts(router, w1, w2, top, bits)
    got = layer(x.cuda()).cpu().double()
    weight, rows, offsets, where = (t.cpu() for t in layer.route(x.cuda()))
    assert int(offsets[0]) == 0 and int(offsets[-1]) == tokens * top and torch.all(offsets[1:] >= offsets[:-1])
    want = torch.zeros(tokens, 256, dtype=torch.float64)
    for t in range(tokens):
        for j in range(top):
            r = int(where[t * top + j])
            assert int(rows[r]) == t
            e = int(torch.searchsorted(offsets, r, right=True)) - 1
            want[t] += float(weight[t, j]) * _plain(x[t:t + 1], w1[e], w2[e], bits)[0]
    assert torch.linalg.norm(got - want) <= 1e-2 * torch.linalg.norm(want)


def test_experts_in_a_graph():
    """The whole layer, routing included, captured once: no step waits for the host."""
    from ptq_int8_lab_b200.mlp import Int8Experts
    rng = np.random.default_rng(1)
    w1, w2 = _weights(rng, 8, 256, 128)
    router = rng.normal(0, 1, (8, 256)).astype(np.float32)
    layer = Int8Experts(router, w1, w2, 2)
    x = torch.zeros((12, 256), device="cuda")
    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
    for seed in range(3):
        x.copy_(torch.from_numpy(np.random.default_rng(seed).normal(0, 1, (12, 256)).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, layer(x))
    del graph


def test_command(capsys):
    from ptq_int8_lab_b200 import mlp
    mlp.main(["--tokens", "7", "--hidden", "128", "--width", "192", "--experts", "4"])
    lines = capsys.readouterr().out.splitlines()
    assert lines[0].startswith("dense: 7 tokens") and lines[1].startswith("experts: top 2 of 4")
    # two quantizations at 8 bits: steps of 1/127 of a row's largest value, uniform errors of a few tenths of a percent
    assert all(float(l.rsplit(" ", 1)[1]) < 0.05 for l in lines)


def test_refusals():
    from ptq_int8_lab_b200.mlp import Int8Experts, lay_weights
    with pytest.raises(E.Ptq8Error, match="bits 3"):
        lay_weights(np.zeros((4, 4), np.float32), 3)
    with pytest.raises(E.Ptq8Error, match="channels, in"):
        lay_weights(np.zeros(4, np.float32))
    with pytest.raises(E.Ptq8Error, match="top 5 of 4"):
        Int8Experts(np.zeros((4, 16)), np.zeros((4, 32, 16)), np.zeros((4, 16, 16)), 5)
