"""A handle that ends before the work it enqueued."""
import numpy as np
import pytest
import torch

from ptq_int8_lab_b200 import engine as E

pytestmark = pytest.mark.gpu


def _operands(rows, k, n):
    rng = np.random.default_rng(rows)
    x = torch.from_numpy(rng.integers(-128, 128, (rows, k), dtype=np.int8)).cuda()
    w = torch.from_numpy(rng.integers(-128, 128, (n, k), dtype=np.int8)).cuda()
    return x, torch.ones(rows, device="cuda"), w, torch.full((n,), 1e-3, device="cuda")


def test_destroyed_while_its_kernels_run():
    """The handle goes while a kernel whose wait will run out waits behind another on the stream: the kernel reports into
    memory that is still there, and no later handle reads that report as its own."""
    from ptq_int8_lab_b200.ops import Int8Ops
    a = _operands(16, 1024, 256)
    want = Int8Ops(0).linear(*a)
    torch.cuda.synchronize()
    ops = Int8Ops(0)
    ops.set_wait_test(10_000_000, True)
    torch.cuda._sleep(50_000_000)
    ops.linear(*a)
    del ops
    others = [Int8Ops(0) for _ in range(4)]
    torch.cuda.synchronize()
    for o in others:
        got = o.linear(*a)
        o.check_device_error()
        assert torch.equal(got, want)


def test_graph_outlives_its_handle():
    from ptq_int8_lab_b200.ops import Int8Ops
    a = _operands(40, 512, 320)
    ops = Int8Ops(0)
    want = ops.linear(*a)
    y = torch.zeros_like(want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.linear(*a, out=y)
    del ops
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    del graph


def test_close():
    """close() reports what the handle's calls left; a closed handle refuses calls, and closes again without a word."""
    from ptq_int8_lab_b200.ops import Int8Ops
    a = _operands(16, 1024, 256)
    ops = Int8Ops(0)
    ops.set_wait_test(10_000_000, True)
    ops.linear(*a)
    with pytest.raises(E.Ptq8Error, match="ran out"):
        ops.close()
    with pytest.raises(E.Ptq8Error, match="null handle"):
        ops.linear(*a)
    ops.close()
    with Int8Ops(0) as ops:
        ops.linear(*a)
    with pytest.raises(E.Ptq8Error, match="null handle"):
        ops.quantize_rows(torch.ones((2, 64), device="cuda"))
    torch.cuda.synchronize()


def test_many_handles():
    """More handles than one block of error words holds, each with its own word."""
    from ptq_int8_lab_b200.ops import Int8Ops
    a = _operands(16, 256, 64)
    bad = None
    for i in range(1100):
        with Int8Ops(0) as ops:
            if i % 100 == 0:
                ops.linear(*a)
        if i == 1000:
            bad = Int8Ops(0)
            bad.set_wait_test(10_000_000, True)
            bad.linear(*a)
    with pytest.raises(E.Ptq8Error, match="ran out"):
        bad.check_device_error()
