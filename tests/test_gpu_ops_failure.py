"""Failure detection of the token operators: a device wait that runs out is reported, and the handle recovers.

The first operand load of the first block is announced to its barrier and never issued; every wait on it is bounded
(about 5 ms here), so the kernel gives up, frees what it holds and returns."""
import numpy as np
import pytest
import torch

from ptq_int8_lab_b200 import engine as E

pytestmark = pytest.mark.gpu

TIMEOUT = 4   # PTQ8_ERR_TIMEOUT


@pytest.mark.parametrize("rows,k,n,bits,act", [(5, 1024, 256, 8, 0), (16, 4096, 4096, 8, 0), (16, 4096, 512, 4, 1),
                                               (100, 512, 300, 8, 1), (600, 1024, 512, 4, 0), (6000, 512, 2048, 8, 0),
                                               (6000, 512, 2048, 4, 1)])
def test_wait_runs_out(rows, k, n, bits, act):
    from ptq_int8_lab_b200.ops import Int8Ops
    ops, other = Int8Ops(0), Int8Ops(0)
    rng = np.random.default_rng(rows)
    ch = n * (2 if act else 1)
    x = torch.from_numpy(rng.integers(-128, 128, (rows, k), dtype=np.int8)).cuda()
    w = torch.from_numpy(rng.integers(0, 256, (ch, k if bits == 8 else k // 2)).astype(np.uint8)).cuda()
    w = w.view(torch.int8) if bits == 8 else w
    xs, ws = torch.ones(rows, device="cuda"), torch.full((ch,), 1e-5, device="cuda")
    good = ops.linear(x, xs, w, ws, bits=bits, act=act)
    ops.check_device_error()
    ops.set_wait_test(10_000_000, True)
    ops.linear(x, xs, w, ws, bits=bits, act=act)
    with pytest.raises(E.Ptq8Error, match="ran out") as e:
        ops.check_device_error()
    assert e.value.status == TIMEOUT
    # another handle never saw it; this one works again once it is reported
    assert torch.equal(other.linear(x, xs, w, ws, bits=bits, act=act), good)
    ops.set_wait_test()
    assert torch.equal(ops.linear(x, xs, w, ws, bits=bits, act=act), good)
    ops.check_device_error()


def test_calls_refused_until_reported():
    from ptq_int8_lab_b200.ops import Int8Ops
    ops = Int8Ops(0)
    x, xs = torch.zeros((6, 64), dtype=torch.int8, device="cuda"), torch.ones(6, device="cuda")
    w, ws = torch.zeros((32, 64), dtype=torch.int8, device="cuda"), torch.ones(32, device="cuda")
    ops.set_wait_test(10_000_000, True)
    ops.linear(x, xs, w, ws)
    torch.cuda.synchronize()
    ops.set_wait_test()
    for call in (lambda: ops.linear(x, xs, w, ws), lambda: ops.quantize_rows(torch.ones((2, 64), device="cuda"))):
        with pytest.raises(E.Ptq8Error, match="earlier call") as e:
            call()
        assert e.value.status == TIMEOUT
    with pytest.raises(E.Ptq8Error):
        ops.check_device_error()
    ops.linear(x, xs, w, ws)
    ops.check_device_error()
