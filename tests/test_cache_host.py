"""The 4-bit cache's and linear_w4's parts that need no GPU: packed structs, null handles, and the 64-bit forms that the GPU tests
compare with, against loops over single numbers."""
import math

import pytest
import torch

from ptq_int8_lab_b200 import engine as E
from tests import cache_reference as R


def test_argument_structs():
    from ptq_int8_lab_b200 import ops
    assert ops._CACHE_ROWS.size == 224 and ops._ATTENTION.size == 248 and ops._W4.size == 112 and ops._WORKSPACE_AT == 216


def test_null_handles():
    L = E.lib()
    for name in ("ptq8_cache_write", "ptq8_cache_read", "ptq8_cache_attention", "ptq8_linear_w4"):
        assert name in E.EXPORTS and getattr(L, name)(None, None, None) == 1
    assert L.ptq8_cache_attention_workspace(None, None) == -1


def test_host_extension_looks_and_leaves():
    """Whatever it does not know it answers with -1, and calls nothing."""
    from ptq_int8_lab_b200 import ops
    host = ops._host_module()
    x = torch.zeros((2, 64))
    for call in (host.linear_w4, host.cache_attention, host.cache_rows):
        assert call() == -1 and call(*[None] * 10) == -1
    assert host.linear_w4(1, 0, x, x, x, 64, None, 0, x, 0) == -1          # tensors of the host
    assert host.linear_w4(1, 0, x, x, x, "64", None, 0, x, 0) == -1
    assert host.linear_w4(1, 0, x, x, x, 64, None, 2 ** 70, x, 0) == -1
    assert host.cache_rows(True, 1, 0, (x, x, x, x), x, x, x, x, None, 0) == -1
    assert host.cache_attention(1, 0, x, [x] * 4, x, x, None, None, x, 0) == -1


@pytest.mark.parametrize("scale", [1.0, 1e-30, 1e30, 0.0])
def test_codes(scale):
    """Every value is within half a step (and a step's own rounding up) of what stands for it."""
    x = (torch.randn((50, 64), generator=torch.Generator().manual_seed(0)) * scale).float()
    codes, step, least = R.quantized(x)
    assert float(codes.min()) >= 0 and float(codes.max()) <= 15
    assert bool((least <= x.double().amin(1, keepdim=True)).all())
    # half a step, and the f32 roundings of x - least and of its quotient: 2^-24 each of at most 16 steps
    assert bool(((least + step * codes - x.double()).abs() <= step * (0.5 + 2 * 16 * 2.0 ** -24)).all())
    # a step is at most a bf16 number above a fifteenth of the spread, which least makes at most 2^-7 of itself wider
    spread = x.double().amax(1, keepdim=True) - least
    assert bool((step <= (spread / 15 * (1 + 2.0 ** -7) * (1 + 2.0 ** -23)).clamp_min(2.0 ** -100)).all())


def test_attention_in_64_bits():
    g = torch.Generator().manual_seed(1)
    page, kv, per, dim, pages = 16, 2, 3, 64, 5
    parts = []
    for _ in range(2):
        parts += [torch.randint(0, 256, (pages, kv, page, dim // 2), generator=g).to(torch.uint8), torch.rand((pages, kv, page, 2), generator=g).to(torch.bfloat16)]
    table = torch.tensor([[3, 0], [4, -1]], dtype=torch.int32)
    lengths, starts = torch.tensor([20, 30], dtype=torch.int32), torch.tensor([0, 2, 3], dtype=torch.int32)
    q = torch.randn((3, kv * per, dim), generator=g).to(torch.bfloat16)
    y, bound = R.attention(q, parts, table, lengths, starts, 0.125, torch.zeros_like(q))
    assert bool((bound >= 0).all())
    for t, (b, pos) in enumerate(((0, 18), (0, 19), (1, 29))):
        for h in range(kv * per):
            terms = []
            for j in range(pos + 1):
                name = int(table[b, j // page])
                if not 0 <= name < pages:
                    continue
                rows = []
                for i in (0, 2):
                    at = parts[i][name, h // per, j % page]
                    s, m = (float(z) for z in parts[i + 1][name, h // per, j % page])
                    rows.append([m + s * (int(at[d // 2]) >> (4 * (d % 2)) & 15) for d in range(dim)])
                terms.append((0.125 * sum(float(a) * c for a, c in zip(q[t, h], rows[0])), rows[1]))
            top = max(z for z, _ in terms)
            total = sum(math.exp(z - top) for z, _ in terms)
            for d in (0, 1, 31, 63):
                want = sum(math.exp(z - top) * v[d] for z, v in terms) / total
                assert abs(float(y[t, h, d]) - want) <= 1e-12 * max(1.0, abs(want))
