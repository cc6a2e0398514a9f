"""The quantized MLPs at sizes where a step has nothing to do."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _weights(rng, experts, hidden, width):
    w1 = (rng.normal(0, 1, (experts, 2 * width, hidden)) / np.sqrt(hidden)).astype(np.float32)
    w2 = (rng.normal(0, 1, (experts, hidden, width)) / np.sqrt(width)).astype(np.float32)
    return w1, w2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
def test_no_tokens(bits, dtype):
    """A batch without tokens, as the end of a request's prompt leaves it."""
    from ptq_int8_lab_b200.mlp import Int8Experts, Int8MLP
    rng = np.random.default_rng(0)
    w1, w2 = _weights(rng, 4, 96, 64)
    x = torch.empty((0, 96), device="cuda", dtype=dtype)
    for layer in (Int8MLP(w1[0], w2[0], bits), Int8Experts(rng.normal(0, 1, (4, 96)), w1, w2, 2, bits)):
        y = layer(x)
        assert y.shape == (0, 96) and y.dtype == dtype
        layer.ops.check_device_error()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("shape", [(5, 33), (3, 7, 40), (2, 2, 3, 1)])
def test_laid_weights_are_quantized_like_the_engine_s(bits, shape):
    """lay_weights itself: quantize_weight's codes and scales, in the layout that the operators take."""
    from ptq_int8_lab_b200 import engine as E
    from ptq_int8_lab_b200.mlp import lay_weights
    w = np.random.default_rng(bits).normal(0, 1, shape).astype(np.float32)
    codes, scale = lay_weights(w, bits)
    want, s = E.quantize_weight(w.reshape(-1, shape[-1]), bits)
    assert codes.is_cuda and codes.dtype == (torch.int8 if bits == 8 else torch.uint8) and codes.stride(-2) % 16 == 0
    assert codes.shape == (*shape[:-1], shape[-1] if bits == 8 else (shape[-1] + 1) // 2) and scale.shape == shape[:-1]
    assert np.array_equal(scale.cpu().numpy().reshape(-1), s)
    got = codes.cpu().numpy().reshape(want.shape[0], -1).astype(np.int16)
    if bits == 4:
        got = np.stack([got & 15, got >> 4], axis=-1).reshape(want.shape[0], -1)[:, :shape[-1]]
        got = np.where(got > 7, got - 16, got)
    assert np.array_equal(got, want)


def _codes(x):
    top = np.abs(x).max()
    s = np.maximum(np.float32(top) / np.float32(127), np.float32(1e-8)).astype(np.float64)
    q = x.astype(np.float64) / s
    return np.sign(q) * np.floor(np.abs(q) + 0.5), s


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens,experts,top", [(1, 4, 2), (33, 8, 2), (40, 5, 5), (7, 16, 1)])
def test_experts_with_routing_of_its_own(bits, tokens, experts, top):
    """The whole layer against a form in numpy that routes by itself: the `top` largest logits of a token, weighted by
    their softmax.  Logits lie a twentieth apart, far more than their 32-bit sums are off.  Codes of the hidden state may
    differ by a step where its value is off in its last places: 1e-2 of a row's norm covers any few (see the layer's tests)."""
    from ptq_int8_lab_b200 import engine as E
    from ptq_int8_lab_b200.mlp import Int8Experts
    hidden, width = 128, 144
    rng = np.random.default_rng(tokens)
    w1, w2 = _weights(rng, experts, hidden, width)
    x = rng.normal(0, 1, (tokens, hidden)).astype(np.float32)
    # a router whose logits for these tokens are a permutation of multiples of 0.05, up to rounding
    wanted = np.stack([rng.permutation(experts) for _ in range(tokens)]) * 0.05
    router = np.linalg.lstsq(x.astype(np.float64), wanted, rcond=None)[0].T.astype(np.float32)
    got = Int8Experts(router, w1, w2, top, bits)(torch.from_numpy(x).cuda()).cpu().numpy()
    quantized = [[tuple(np.asarray(v, np.float64) for v in E.quantize_weight(w[e], bits)) for w in (w1, w2)] for e in range(experts)]
    want = np.zeros((tokens, hidden))
    for t in range(tokens):
        chosen = np.argsort(-wanted[t])[:top]
        p = np.exp(wanted[t][chosen])
        c, s = _codes(x[t])
        for e, weight in zip(chosen, p / p.sum()):
            (c1, s1), (c2, s2) = quantized[e]
            z = (c1 @ c) * s * s1
            g, u = z[:width], z[width:]
            ch, sh = _codes((g / (1 + np.exp(-g)) * u).astype(np.float32))
            want[t] += weight * ((c2 @ ch) * sh * s2)
    assert np.linalg.norm(got - want) <= 1e-2 * np.linalg.norm(want)


def test_command_returns_what_it_prints(capsys):
    from ptq_int8_lab_b200 import mlp
    far = mlp.main(["--tokens", "9", "--hidden", "128", "--width", "160", "--experts", "4"])
    printed = [float(line.rsplit(" ", 1)[1]) for line in capsys.readouterr().out.splitlines()]
    assert len(far) == 2 and all(0 < d < 0.05 for d in far)
    assert all(abs(d - p) <= 5.1e-5 for d, p in zip(far, printed))
