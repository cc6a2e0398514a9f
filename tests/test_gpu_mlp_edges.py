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
