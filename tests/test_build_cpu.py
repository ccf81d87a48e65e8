"""CPU: the library is built with or without torch, and the host module again for another Python or torch."""
from __future__ import annotations

import importlib.util
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent


@pytest.fixture
def kb_build(tmp_path, monkeypatch):
    """build.py with its products in tmp_path; compilers are noted, not run, and leave empty files."""
    spec = importlib.util.spec_from_file_location("kb_build_under_test", REPO / "kernelbench-hip_b200" / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.BUILD, mod.LIB = tmp_path / "build", tmp_path / "libkbb200.so"
    mod.HOST_MODULE, mod.HOST_FOR = tmp_path / "_lm_host.so", tmp_path / "build" / "lm_host.for"
    mod.ran = []

    def run(cmd, **_):
        mod.ran.append(Path(cmd[0]).name)
        Path(cmd[cmd.index("-o") + 1]).touch()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(mod.subprocess, "run", run)
    return mod


def without_torch(monkeypatch):
    real = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else real(name, *a))


def test_without_torch(kb_build, monkeypatch, capsys):
    without_torch(monkeypatch)
    assert kb_build.build() == kb_build.LIB and kb_build.LIB.exists() and not kb_build.HOST_MODULE.exists()
    assert "g++" not in kb_build.ran and "torch" in capsys.readouterr().err


def test_library_before_a_host_module_that_fails(kb_build, monkeypatch):
    run = kb_build.subprocess.run

    def fails(cmd, **k):
        if Path(cmd[0]).name == "g++":
            return subprocess.CompletedProcess(cmd, 1, "", "no such header")
        return run(cmd, **k)

    monkeypatch.setattr(kb_build.subprocess, "run", fails)
    with pytest.raises(RuntimeError, match="no such header"):
        kb_build.build()
    assert kb_build.LIB.exists()


def test_host_module_for_another_torch(kb_build, tmp_path, monkeypatch):
    pytest.importorskip("torch")
    kb_build.build()
    assert kb_build.ran.count("g++") == 1
    kb_build.build()
    assert kb_build.ran.count("g++") == 1  # up to date
    # an older installation of another version, as files come out of an archive
    other = tmp_path / "site" / "torch"
    other.mkdir(parents=True)
    (other / "__init__.py").touch()
    (other / "version.py").write_text("__version__ = '1.0'\n")
    spec = importlib.util.spec_from_file_location("torch", other / "__init__.py")
    real = importlib.util.find_spec
    with monkeypatch.context() as m:
        m.setattr(importlib.util, "find_spec", lambda name, *a: spec if name == "torch" else real(name, *a))
        kb_build.build()
        assert kb_build.ran.count("g++") == 2
        kb_build.build()
        assert kb_build.ran.count("g++") == 2
    kb_build.build()
    assert kb_build.ran.count("g++") == 3
