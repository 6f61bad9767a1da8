"""When the extension module beside the library is built, and when it is not: nothing is compiled here."""
import subprocess
import sys
import types
from pathlib import Path

import pytest

from halo_flash_b200 import build


@pytest.fixture
def bind(tmp_path, monkeypatch):
    """_build_bind with a torch of the test's own and a compiler that only counts; returns how often it ran."""
    torch = tmp_path / "torch"
    torch.mkdir()
    (torch / "version.py").write_text("__version__ = '1'\n")
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text("module")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "BIND", tmp_path / "_bind.so")
    monkeypatch.setattr(build, "OBJ", tmp_path)
    monkeypatch.setattr(build, "find_spec", lambda name: types.SimpleNamespace(submodule_search_locations=[str(torch)]))
    monkeypatch.setattr(build.subprocess, "run", run)

    def times(force=False):
        ran.clear()
        build._build_bind("/usr/local/cuda/bin/nvcc", force)
        return len(ran)

    times.torch = torch
    return times


def test_module_is_rebuilt_when_torch_changes(bind, monkeypatch):
    assert bind() == 1 and bind() == 0
    (bind.torch / "version.py").write_text("__version__ = '2'\n")
    assert bind() == 1 and bind() == 0
    monkeypatch.setattr(sys, "version", sys.version + " (another)")
    assert bind() == 1 and bind() == 0
    assert bind(force=True) == 1


def test_library_alone_is_built_without_torch(bind, monkeypatch, capsys):
    monkeypatch.setattr(build, "find_spec", lambda name: None)
    assert bind() == 0 and "no torch" in capsys.readouterr().err


def test_library_alone_is_built_without_python_headers(bind, monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path / "none")})
    assert bind() == 0 and "Python.h" in capsys.readouterr().err


def test_a_failed_module_is_an_error(bind, monkeypatch):
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: subprocess.CompletedProcess(cmd, 1, "", "no such header"))
    with pytest.raises(RuntimeError, match="no such header"):
        bind()
