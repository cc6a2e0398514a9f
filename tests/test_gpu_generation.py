"""The 4-bit operators together, as a layer of a generating model uses them: against the same layer from its parts in 64 bits,
in a captured step, on other streams, and through the commands."""
import math

import numpy as np
import pytest
import torch

from ptq_int8_lab_b200 import engine as E
from tests import cache_reference as R

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, GROUP, PAGE = 256, 6, 2, 64, 64, 16


def weights(seed):
    rng = np.random.default_rng(seed)
    qkv = (rng.normal(0, 1, ((HEADS + 2 * KV) * DIM, HIDDEN)) / math.sqrt(HIDDEN)).astype(np.float32)
    out = (rng.normal(0, 1, (HIDDEN, HEADS * DIM)) / math.sqrt(HEADS * DIM)).astype(np.float32)
    return qkv, out


def stands_for(codes, scale, group):
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(1).double()
    return torch.where(c > 7, c - 16, c) * scale.double().repeat_interleave(group, 1)[:, :c.shape[1]]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_layer():
    """Prompts, then pieces, then single tokens: each output within the roundings of bf16 states and outputs of a 64-bit layer that
    has the layer's own weights and cache."""
    from ptq_int8_lab_b200.attention import Int4Attention
    qkv, out = weights(0)
    layer = Int4Attention(qkv, out, HEADS, KV, 40, PAGE, GROUP)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    table = torch.randperm(40, generator=g, device="cuda").to(torch.int32).view(4, 10)
    lengths = [0, 0, 0, 0]
    w1, w2 = stands_for(*layer.qkv, GROUP), stands_for(*layer.out, GROUP)
    half = 2.0 ** -8   # bf16 keeps 8 places: values in [1, 2) stand 2^-7 apart, and a rounding is off by at most half of that
    for news in ([33, 0, 1, 90], [5, 20, 1, 3], [1, 1, 1, 1], [1, 1, 1, 1]):
        lengths = [a + b for a, b in zip(lengths, news)]
        x = torch.randn((sum(news), HIDDEN), generator=g, device="cuda").to(torch.bfloat16)
        starts = None if news == [1] * 4 else ints([sum(news[:i]) for i in range(5)])
        y = layer(x, table, ints(lengths), starts)
        layer.ops.check_device_error()
        # queries as the layer rounds them; the cache as it is (its codes are tested elsewhere)
        both = layer.ops.linear_w4(x, *layer.qkv, GROUP).view(-1, HEADS + 2 * KV, DIM)
        exact = (x.double() @ w1.t()).view_as(both)
        assert float(((both.double() - exact).abs() / (exact.abs() * half + 1e-3 * half * x.double().norm(dim=1)[:, None, None])).max()) <= 1.0
        att, bound = R.attention(both[:, :HEADS], layer.cache, table, ints(lengths), starts, DIM ** -0.5, torch.zeros_like(both[:, :HEADS]))
        want = att.reshape(-1, HEADS * DIM) @ w2.t()
        # the attention's bound (its rounding to bf16 in it) through the last product, then the output's rounding and f32 sums
        allowed = bound.reshape(-1, HEADS * DIM) @ w2.abs().t() + half * want.abs() + 2.0 ** -16 * (att.abs().reshape(-1, HEADS * DIM) @ w2.abs().t())
        assert float(((y.double() - want).abs() / allowed).max()) <= 1.0
    assert lengths == [40, 22, 4, 95]


def test_captured_step():
    """One graph of a step, replayed while lengths grow on the device and pages fill, gives what eager steps give."""
    from ptq_int8_lab_b200.attention import Int4Attention
    qkv, out = weights(2)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    eager, captured = (Int4Attention(qkv, out, HEADS, KV, 12, PAGE, GROUP) for _ in range(2))
    table = torch.randperm(12, generator=g, device="cuda").to(torch.int32).view(3, 4)
    states = [torch.randn((3, HIDDEN), generator=g, device="cuda").to(torch.bfloat16) for _ in range(40)]
    x, lengths, first = torch.zeros_like(states[0]), ints([0, 7, 15]), ints([0, 7, 15])
    captured(x, table, lengths)   # (loads kernels; overwritten below)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lengths += 1
        y = captured(x, table, lengths)
    lengths.copy_(first)
    for c in (eager.cache, captured.cache):
        for t in c:
            t.zero_()
    now = first.clone()
    for s in states:
        x.copy_(s)
        graph.replay()
        now += 1
        assert torch.equal(y, eager(s, table, now))
    assert torch.equal(lengths, now)
    assert all(torch.equal(a, b) for a, b in zip(eager.cache, captured.cache))
    eager.ops.check_device_error(), captured.ops.check_device_error()
    del graph


def test_two_graphs_at_once():
    """Two captured calls, each with the workspace of its own capture, replayed on two streams at the same time."""
    from ptq_int8_lab_b200.ops import Int8Ops
    from tests.test_gpu_cache import generator, layout, random_cache
    ops = Int8Ops(0)
    g = generator(4)
    work = []
    for lengths in ([5000, 20], [900, 3000]):
        pages, table = layout(g, lengths, 64)
        cache = random_cache(g, pages, 2, 64, 128)
        q = torch.randn((2, 16, 128), generator=g, device="cuda").to(torch.bfloat16)
        n = ints(lengths)
        want = ops.cache_attention(q, cache, table, n)
        torch.cuda.synchronize()
        graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(q)
        with torch.cuda.graph(graph):
            for _ in range(20):
                ops.cache_attention(q, cache, table, n, out=out)
        work.append((graph, torch.cuda.Stream(), out, want, (q, cache, table, n)))
    for _ in range(5):
        for _, _, out, _, _ in work:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream, _, _, _ in work:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, _, out, want, _ in work)
    ops.check_device_error()
    work.clear()


def test_streams():
    """Calls on a stream that is given (workspace and outputs too), and on the current one of another thread of work."""
    from ptq_int8_lab_b200.ops import Int8Ops
    from tests.test_gpu_cache import generator, layout, random_cache
    ops = Int8Ops(0)
    g = generator(5)
    pages, table = layout(g, [3000, 100], 64)
    cache = random_cache(g, pages, 2, 64, 64)
    q = torch.randn((2, 8, 64), generator=g, device="cuda").to(torch.float16)
    n = ints([3000, 100])
    want = ops.cache_attention(q, cache, table, n)
    w, s = torch.randint(0, 256, (96, 64), generator=g, device="cuda").to(torch.uint8), torch.rand((96, 1), generator=g, device="cuda")
    x = torch.randn((2, 128), generator=g, device="cuda")
    want_w = ops.linear_w4(x, w, s, 128)
    need = ops.cache_attention_workspace(q, cache, table, n)
    assert need > 0
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out, workspace, y = torch.zeros_like(q), torch.empty(need, dtype=torch.uint8, device="cuda"), torch.zeros_like(want_w)
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream):
        ops.cache_attention(q, cache, table, n, out=out, workspace=workspace, stream=stream)
        ops.linear_w4(x, w, s, 128, out=y, stream=stream)
        side.synchronize()
        assert torch.equal(out, want) and torch.equal(y, want_w)
        out.zero_(), y.zero_()
    with torch.cuda.stream(side):
        got, got_w = ops.cache_attention(q, cache, table, n), ops.linear_w4(x, w, s, 128)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got_w, want_w)
    k = torch.randn((2, 2, 64), generator=g, device="cuda")
    ops.cache_write(cache, k, k, table, n, stream=side)
    back = [torch.zeros((2, 2, 64), device="cuda") for _ in range(2)]
    side.synchronize()
    ops.cache_read(cache, table, n, out=back, stream=side)
    side.synchronize()
    codes, step, least = R.quantized(k)
    assert all(torch.equal(t.double(), (least + step * codes).float().double()) for t in back)
    for call in (lambda: ops.cache_attention(q, cache, table, n, stream=side), lambda: ops.cache_attention(q, cache, table, n, out=out, stream=side),
                 lambda: ops.linear_w4(x, w, s, 128, stream=side), lambda: ops.cache_read(cache, table, n, stream=side)):
        with pytest.raises(E.Ptq8Error, match="with stream"):
            call()
    ops.check_device_error()


@pytest.mark.parametrize("dim,per,lengths,news", [(128, 4, [3000], None), (64, 16, [300, 20], None), (256, 2, [100], None), (128, 4, [600], [200]), (64, 64, [90], [80]), (64, 64, [1400], [1300])])
def test_attention_s_wait_runs_out(dim, per, lengths, news):
    from ptq_int8_lab_b200.ops import Int8Ops
    from tests.test_gpu_cache import begins, generator, layout, random_cache
    ops, g = Int8Ops(0), generator(6)
    pages, table = layout(g, lengths, 64)
    cache = random_cache(g, pages, 2, 64, dim)
    q = torch.randn((sum(news or [1] * len(lengths)), 2 * per, dim), generator=g, device="cuda").to(torch.bfloat16)
    args = (q, cache, table, ints(lengths), begins(news) if news else None)
    good = ops.cache_attention(*args)
    ops.check_device_error()
    ops.set_wait_test(10_000_000, True)
    ops.cache_attention(*args)
    with pytest.raises(E.Ptq8Error, match="ran out") as e:
        ops.check_device_error()
    assert e.value.status == 4
    ops.set_wait_test()
    assert torch.equal(ops.cache_attention(*args), good)
    ops.check_device_error()


@pytest.mark.parametrize("tokens,inp,out,group,gated", [(8, 4096, 512, 128, False), (5, 256, 40, 32, True), (40, 2048, 2000, 64, False), (3, 20000, 64, 128, True)])
def test_linear_w4_s_wait_runs_out(tokens, inp, out, group, gated):
    from ptq_int8_lab_b200.ops import Int8Ops
    ops = Int8Ops(0)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    w = torch.randint(0, 256, (out * (1 + gated), inp // 2), generator=g, device="cuda").to(torch.uint8)
    s = torch.rand((w.shape[0], -(-inp // group)), generator=g, device="cuda")
    x = torch.randn((tokens, inp), generator=g, device="cuda").to(torch.bfloat16)
    good = ops.linear_w4(x, w, s, group, act=int(gated))
    ops.check_device_error()
    ops.set_wait_test(10_000_000, True)
    ops.linear_w4(x, w, s, group, act=int(gated))
    with pytest.raises(E.Ptq8Error, match="ran out") as e:
        ops.check_device_error()
    assert e.value.status == 4
    ops.set_wait_test()
    assert torch.equal(ops.linear_w4(x, w, s, group, act=int(gated)), good)
    ops.check_device_error()


def test_closed_handle():
    from ptq_int8_lab_b200.ops import Int8Ops, new_cache
    ops = Int8Ops(0)
    cache = new_cache(1, 1, 64, 16)
    x, w, s = torch.zeros((1, 64), device="cuda"), torch.zeros((8, 32), dtype=torch.uint8, device="cuda"), torch.ones((8, 1), device="cuda")
    k, table, n = torch.zeros((1, 1, 64), device="cuda"), ints([[0]]), ints([1])
    ops.close()
    q = k.to(torch.float16)
    for call in (lambda: ops.linear_w4(x, w, s, 64), lambda: ops.linear_w4(x, w, s, 64, out=torch.zeros((1, 8), device="cuda")),
                 lambda: ops.cache_write(cache, k, k, table, n), lambda: ops.cache_read(cache, table, n), lambda: ops.cache_attention(q, cache, table, n)):
        with pytest.raises(E.Ptq8Error, match="null handle"):
            call()


def test_commands():
    from ptq_int8_lab_b200 import attention, mlp
    far = attention.main(["--sequences", "3", "--prompt", "70", "--steps", "3", "--hidden", "256", "--heads", "4", "--kv-heads", "2"])
    assert all(0.0 < d < 1.0 for d in far), far   # it runs, and NaN fails
    far = mlp.main(["--tokens", "6", "--hidden", "128", "--width", "192", "--experts", "2", "--group", "32"])
    assert len(far) == 3 and all(0.0 < d < 1.0 for d in far), far
