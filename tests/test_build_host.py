"""The build and the Python extension: the library is made without torch, and in spite of an extension that does not compile."""
import subprocess
import sys
from pathlib import Path

import pytest

from ptq_int8_lab_b200 import build as B
from ptq_int8_lab_b200 import engine as E


@pytest.fixture
def compilers(tmp_path, monkeypatch):
    """Compilers that write their output, and fail where its name is in the set that this gives."""
    failing = set()

    class Compiler:
        def __init__(self, cmd):
            self.out = Path(cmd[cmd.index("-o") + 1])

        def wait(self):
            if self.out.name in failing:
                return 1
            self.out.write_text("x")
            return 0
    monkeypatch.setattr(B, "OUT", tmp_path)
    monkeypatch.setattr(B, "HOST", tmp_path / "ptq8_host.so")
    monkeypatch.setattr(subprocess, "Popen", Compiler)
    monkeypatch.setattr(subprocess, "check_call", lambda cmd: Compiler(cmd).wait())
    return failing


def test_without_torch(compilers, tmp_path, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)   # (import torch raises)
    assert B.build() == tmp_path / "libptq8.so"
    assert sorted(p.name for p in tmp_path.iterdir()) == ["libptq8.so"]


def test_with_torch(compilers, tmp_path):
    B.build()
    assert sorted(p.name for p in tmp_path.iterdir()) == ["libptq8.so", "ptq8_host.so"]


def test_an_extension_that_does_not_compile(compilers, tmp_path):
    """The library is there; the build says what failed."""
    compilers.add("ptq8_host.so.tmp")
    with pytest.raises(subprocess.CalledProcessError, match="ptq8_host"):
        B.build()
    assert sorted(p.name for p in tmp_path.iterdir()) == ["libptq8.so"]


def test_a_library_that_does_not_compile(compilers, tmp_path):
    compilers.add("ptq8_ops.o")
    with pytest.raises(subprocess.CalledProcessError, match="ptq8_ops"):
        B.build()
    assert not (tmp_path / "libptq8.so").exists()


def test_an_extension_that_is_not_there_or_does_not_load(tmp_path, monkeypatch):
    from ptq_int8_lab_b200 import ops
    monkeypatch.setattr(ops, "_host", None)
    monkeypatch.setattr(B, "HOST", tmp_path / "ptq8_host.so")
    with pytest.raises(E.Ptq8Error, match="not found: build it"):
        ops._host_module()
    (tmp_path / "ptq8_host.so").write_bytes(b"not a library")
    with pytest.raises(E.Ptq8Error, match="does not fit"):
        ops._host_module()


@pytest.mark.gpu
def test_operators_that_do_without_it(tmp_path, monkeypatch):
    """quantize_rows and linear run where the extension is missing; the others say what is missing, and make up for it once it is there."""
    import torch
    from ptq_int8_lab_b200 import ops
    here = B.HOST
    monkeypatch.setattr(ops, "_host", None)
    monkeypatch.setattr(B, "HOST", tmp_path / "ptq8_host.so")
    with ops.Int8Ops(0) as o:
        x = torch.randn((4, 64), device="cuda")
        codes, scale = o.quantize_rows(x)
        w, ws = torch.ones((8, 64), dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
        assert o.linear(codes, scale, w, ws, dtype=torch.float32).shape == (4, 8)
        cache = ops.new_cache(1, 1, 64, 16)
        k = torch.randn((1, 1, 64), device="cuda")
        table, lengths = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
        with pytest.raises(E.Ptq8Error, match="not found"):
            o.cache_write(cache, k, k, table, lengths)
        monkeypatch.setattr(B, "HOST", here)
        o.cache_write(cache, k, k, table, lengths)
        assert cache.k.any()
        o.check_device_error()
