"""The build script, with the compilers replaced: what it makes where there is no PyTorch."""

import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(monkeypatch, tmp_path):
    """cc1d_build writing into tmp_path; .calls are the compilers' command lines."""
    monkeypatch.syspath_prepend(os.path.join(ROOT, "cute-causal-conv1d_b200"))
    import cc1d_build

    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(cc1d_build, "BUILD", str(tmp_path / "objects"))
    monkeypatch.setattr(cc1d_build, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(cc1d_build, "BINDING", str(tmp_path / "binding.so"))
    monkeypatch.setattr(cc1d_build, "nvcc", lambda: "/cuda/bin/nvcc")
    monkeypatch.setattr(cc1d_build.subprocess, "run", run)
    cc1d_build.calls = calls
    return cc1d_build


def test_library_alone_without_torch(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    build.build()
    assert os.path.exists(build.LIB) and not os.path.exists(build.BINDING)
    assert all(c[0] == "/cuda/bin/nvcc" for c in build.calls) and len(build.calls) == len(build.UNITS) + 1
    assert "_block.so is not built" in capsys.readouterr().err
    assert build.up_to_date()
    build.build()
    assert len(build.calls) == len(build.UNITS) + 1  # nothing to do


def test_binding_follows_when_torch_is_there(build):
    build.build()
    assert os.path.exists(build.LIB) and os.path.exists(build.BINDING) and build.up_to_date()
    os.remove(build.BINDING)
    assert not build.up_to_date()


def test_a_binding_that_does_not_compile_leaves_the_library(build, monkeypatch):
    def broken(obj):
        raise RuntimeError("g++ failed")

    monkeypatch.setattr(build, "compile_binding", broken)
    with pytest.raises(RuntimeError, match="g\\+\\+ failed"):
        build.build()
    assert os.path.exists(build.LIB) and not os.path.exists(build.BINDING)
