"""Weights laid in groups: sizes of groups beyond a row's."""
import numpy as np
import pytest
import torch

from ptq_int8_lab_b200 import engine as E

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [100, 101, 128, 1 << 20, 1 << 31, 1 << 40])
def test_a_group_of_all_features_and_more(group):
    """One scale a row, the same codes, and no more memory than the row takes."""
    from ptq_int8_lab_b200.mlp import lay_groups, lay_weights
    w = np.random.default_rng(0).normal(0, 1, (6, 100)).astype(np.float32)
    codes, scale = lay_groups(w, group)
    want, one = lay_weights(w, 4)
    assert codes.shape == (6, 50) and codes.stride(0) == 64 and scale.shape == (6, 1)
    assert torch.equal(codes, want) and torch.equal(scale[:, 0], one)


@pytest.mark.parametrize("group", [0, -32])
def test_refused_groups(group):
    from ptq_int8_lab_b200.mlp import lay_groups
    with pytest.raises(E.Ptq8Error, match="group"):
        lay_groups(np.zeros((2, 8), dtype=np.float32), group)


def test_a_layer_with_one_group_a_row():
    from ptq_int8_lab_b200.mlp import Int4MLP
    rng = np.random.default_rng(1)
    gate_up, down = rng.normal(0, 0.1, (256, 96)).astype(np.float32), rng.normal(0, 0.1, (96, 128)).astype(np.float32)
    x = torch.randn((5, 96), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    want = Int4MLP(gate_up, down, 128)(x)
    assert torch.equal(Int4MLP(gate_up, down, 1 << 30)(x), want)
