"""The Python extension's calls run without the interpreter's lock, and hold their tensors meanwhile."""
import ctypes
import importlib.util
import shutil
import threading
import time

import pytest
import torch

from tests.test_gpu_cache import generator, ints, random_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def slow(tmp_path_factory):
    """The extension once more, its entry points a C function that sleeps as many microseconds as the handle's number says."""
    from ptq_int8_lab_b200.build import HOST
    copy = tmp_path_factory.mktemp("host") / "ptq8_host.so"
    shutil.copy(HOST, copy)
    spec = importlib.util.spec_from_file_location("ptq8_host", copy)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    libc = ctypes.CDLL(None)
    usleep, labs = (ctypes.cast(f, ctypes.c_void_p).value for f in (libc.usleep, libc.labs))   # labs: a workspace of so many bytes
    module.entries(usleep, usleep, usleep, labs, usleep)
    return module


def calls(module):
    g = generator(0)
    cache = random_cache(g, 4, 2, 16, 64)
    k = torch.zeros((3, 2, 64), device="cuda")
    q = torch.zeros((3, 4, 64), dtype=torch.float16, device="cuda")
    table, lengths = ints([[0], [1], [2]]), ints([5, 6, 7])
    x, w, s = torch.zeros((2, 64), device="cuda"), torch.zeros((8, 32), dtype=torch.uint8, device="cuda"), torch.ones((8, 1), device="cuda")
    y = torch.zeros((2, 8), device="cuda")
    return {"write": lambda us, c: module.cache_rows(True, us, 0, c, k, k, table, lengths, None, 0),
            "read": lambda us, c: module.cache_rows(False, us, 0, c, k, k.clone(), table, lengths, None, 0),
            "attention": lambda us, c: module.cache_attention(us, 0, q, c, table, lengths, None, None, q.clone(), 0),
            "linear": lambda us, c: module.linear_w4(us, 0, x, w, s, 64, None, 0, y, 0)}, cache


@pytest.mark.parametrize("name", ["write", "read", "attention", "linear"])
def test_other_threads_go_on(slow, name):
    made, cache = calls(slow)
    assert made[name](1, cache) == 0
    ticks, done = [], threading.Event()

    def tick():
        while not done.is_set():
            ticks.append(time.perf_counter())
            time.sleep(0.001)
    other = threading.Thread(target=tick)
    other.start()
    try:
        begin = time.perf_counter()
        assert made[name](400_000, cache) == 0
        end = time.perf_counter()
    finally:
        done.set()
        other.join()
    assert end - begin >= 0.39
    assert sum(begin + 0.1 < t < begin + 0.3 for t in ticks) >= 10


@pytest.mark.parametrize("name", ["write", "read", "attention"])
def test_tensors_are_held(slow, name):
    """A list of the cache's tensors that another thread empties during the call: they stay until it is over."""
    made, cache = calls(slow)
    parts = list(cache)
    del cache

    def empty():
        time.sleep(0.1)
        parts.clear()
    other = threading.Thread(target=empty)
    other.start()
    before = torch.cuda.memory_allocated()
    seen = []

    def look():
        time.sleep(0.2)
        seen.append(torch.cuda.memory_allocated())
    third = threading.Thread(target=look)
    third.start()
    assert made[name](400_000, parts) == 0
    other.join(), third.join()
    assert not parts
    assert seen[0] >= before and torch.cuda.memory_allocated() < seen[0]
