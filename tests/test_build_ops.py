"""The module behind moonshine_amd.ops is built for one torch: another torch means another module, and without torch's headers the rest still builds."""
import os
import sys
import time
import types

import pytest
import torch

from moonshine_amd import build, ops


def test_module_says_which_torch_it_was_built_for():
    assert ops._ops.torch_version == torch.__version__


@pytest.fixture
def compiler(tmp_path, monkeypatch):
    """build_ops() with a compiler that only notes that it was called, and a library folder of its own."""
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("module")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build, "LIB_OPS", str(tmp_path / "msh_torch_ops.so"))
    monkeypatch.setattr(build.subprocess, "run", run)
    return calls


def test_another_torch_builds_another_module(compiler, monkeypatch):
    build.build_ops()
    assert len(compiler) == 1
    future = time.time() + 60
    os.utime(build.LIB_OPS, (future, future))
    build.build_ops()
    assert len(compiler) == 1                                 # nothing changed
    monkeypatch.setattr(torch, "__version__", "9.9.9+other")
    build.build_ops()
    assert len(compiler) == 2


def test_the_library_builds_without_torch(compiler, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)           # (import torch raises)
    assert build.build_ops() is None and not compiler
    assert "moonshine_amd.ops" in capsys.readouterr().err


def test_the_library_builds_without_torchs_headers(compiler, monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(torch, "__file__", str(tmp_path / "__init__.py"))
    assert build.build_ops() is None and not compiler
    assert "headers" in capsys.readouterr().err


def test_a_module_of_another_torch_is_not_used(monkeypatch):
    monkeypatch.setattr(torch, "__version__", "9.9.9+other")
    with pytest.raises(ImportError, match="built for torch"):
        ops._load()
