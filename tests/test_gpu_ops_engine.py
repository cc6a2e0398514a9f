"""Token operators and the engine's forward passes on one stream, launch after launch: both start while the kernel before
them drains, and both hold TMEM."""
import numpy as np
import pytest
import torch

from ptq_int8_lab_b200 import engine as E

pytestmark = pytest.mark.gpu


def _product(rng, rows, k, n, bits):
    x = torch.from_numpy(rng.integers(-128, 128, (rows, k), dtype=np.int8)).cuda()
    w = torch.from_numpy(rng.integers(0, 256, (n, k * bits // 8)).astype(np.uint8)).cuda()
    return x, torch.ones(rows, device="cuda"), w.view(torch.int8) if bits == 8 else w, torch.full((n,), 1e-3, device="cuda")


def test_one_stream(make_model):
    """Convolutions of all sizes between products of all kinds: outputs are those of each alone."""
    from ptq_int8_lab_b200.ops import Int8Ops
    p = make_model(0)
    ops = Int8Ops(0)
    rng = np.random.default_rng(0)
    n = 16
    eng = E.open_engine(p["model"], p["calib"], p["plan"], max_batch=n)
    x = rng.standard_normal((n, 3, 32, 32)).astype(np.float32)
    want = eng.forward(x)
    xd = torch.from_numpy(x).cuda()
    # one tile a group of CTAs, split sums, tiles of every size, pairs; both weight types
    calls = [(_product(rng, rows, k, ch, bits), bits) for rows, k, ch in ((9, 4096, 512), (64, 1024, 4096), (130, 512, 2048), (2000, 512, 4096))
             for bits in (8, 4)]
    alone = [ops.linear(*a, bits=bits) for a, bits in calls]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    eng.set_stream(stream.cuda_stream)
    logits = [torch.empty(n, want.shape[1], device="cuda") for _ in range(10)]
    outs = [torch.empty_like(y) for y in alone]
    torch.cuda.synchronize()
    for ld in logits:
        for (a, bits), y in zip(calls, outs):
            ops.linear(*a, bits=bits, out=y, stream=stream)
            ops.linear(*a, bits=bits, out=y, stream=stream)
            eng.forward_device(xd.data_ptr(), n, ld.data_ptr())
    ops.check_device_error(stream)
    eng.sync()
    for y, z in zip(outs, alone):
        assert torch.equal(y, z)
    for ld in logits:
        assert np.array_equal(ld.cpu().numpy(), want)
