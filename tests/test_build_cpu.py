"""The build's optional part: the compiled Python entry points need torch, the C library does
not."""
import builtins
import importlib.util
import os
import sys
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent / "fused-moe-yws_b200"


@pytest.fixture
def builder(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("fmoe_build", ROOT / "build.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    commands = []

    def run(cmd, *a, **k):
        commands.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_bytes(b"")

    monkeypatch.setattr(m, "LIB", tmp_path)
    monkeypatch.setattr(m.subprocess, "check_call", run)
    m.commands = commands
    return m


def test_build_without_torch_makes_the_library(builder, monkeypatch, capsys):
    """The core is built and the binding left out, with a line that says so."""
    real = builtins.__import__

    def no_torch(name, *a, **k):
        if name == "torch" or name.startswith("torch."):
            raise ModuleNotFoundError("No module named 'torch'", name="torch")
        return real(name, *a, **k)

    monkeypatch.setattr(builder, "build_core", lambda verbose=False: Path("core"))
    monkeypatch.setattr(builder, "build_tvm_ffi", lambda verbose=False: None)
    monkeypatch.delitem(sys.modules, "torch")
    monkeypatch.setattr(builtins, "__import__", no_torch)
    assert builder.build() == (Path("core"), None)
    assert not builder.commands
    assert "fmoe_torch.so" in capsys.readouterr().out


def test_build_without_the_headers_of_torch(builder, tmp_path, monkeypatch):
    """A torch without C++ headers, or without CUDA libraries, is no torch to build against."""
    monkeypatch.setattr(torch, "__file__", str(tmp_path / "torch" / "__init__.py"))
    assert builder.build_torch() is None and not builder.commands


def test_binding_is_rebuilt_for_another_torch(builder, tmp_path, monkeypatch):
    so = tmp_path / "fmoe_torch.so"
    assert builder.build_torch() == so and len(builder.commands) == 1
    os.utime(so)
    assert builder.build_torch() == so and len(builder.commands) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1+other")
    assert builder.build_torch() == so and len(builder.commands) == 2
    assert builder.build_torch() == so and len(builder.commands) == 2


def test_binding_of_another_torch_is_not_loaded(fmoe, monkeypatch):
    from fmoe_b200 import router

    monkeypatch.setattr(router, "_module", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1+other")
    with pytest.raises(RuntimeError, match="0.0.1.other"):
        fmoe.route_experts(torch.zeros(4, 8), 2)
