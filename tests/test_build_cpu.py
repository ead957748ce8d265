"""The build command where only nvcc is there: a C host needs neither torch nor Python's headers."""

from __future__ import annotations

import importlib.util
import sys
import sysconfig

import pytest

from conftest import REPO


@pytest.fixture
def build(monkeypatch, tmp_path):
    """build.py with its library up to date, and the Python side to be built under tmp_path."""
    spec = importlib.util.spec_from_file_location("q3_build",
                                                  REPO / "qwen3-tile-ops_b200" / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    obj = tmp_path / "a.o"
    obj.touch()
    monkeypatch.setattr(mod, "_compile", lambda src, verbose: obj)
    monkeypatch.setattr(mod, "LIB", tmp_path / "libq3b200.so")
    monkeypatch.setattr(mod, "NATIVE", tmp_path / "_native.so")
    mod.LIB.touch()
    return mod


def test_build_without_torch(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build() == build.LIB
    assert "torch" in capsys.readouterr().err and not build.NATIVE.exists()


def test_build_without_python_headers(build, monkeypatch, capsys, tmp_path):
    pytest.importorskip("torch")
    paths = dict(sysconfig.get_paths(), include=str(tmp_path / "none"))
    monkeypatch.setattr(sysconfig, "get_paths", lambda: paths)
    assert build.build() == build.LIB
    assert "Python.h" in capsys.readouterr().err and not build.NATIVE.exists()


def test_build_reports_a_compiler_that_fails(build, monkeypatch):
    pytest.importorskip("torch")
    monkeypatch.setenv("CXX", "false")
    with pytest.raises(RuntimeError, match="_native.so"):
        build.build()
