"""CPU tests of forge_amd.build: the C library needs hipcc alone."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

from forge_amd import build


def test_without_torch_there_is_no_binding_and_no_error(monkeypatch, tmp_path, capsys):
    old = tmp_path / "_step.so"
    old.write_bytes(b"of an earlier library")
    monkeypatch.setattr(build, "STEP", str(old))
    monkeypatch.setitem(sys.modules, "torch", None)
    build._binding()
    assert not old.exists()  # (it would call the new library by the old one's header)
    assert "torch" in capsys.readouterr().out


def test_without_a_host_compiler_there_is_no_binding_and_no_error(monkeypatch, tmp_path, capsys):
    pytest.importorskip("torch")
    monkeypatch.setattr(build, "STEP", str(tmp_path / "_step.so"))
    monkeypatch.setenv("PATH", str(tmp_path))
    build._binding()
    assert not os.listdir(tmp_path) and "g++" in capsys.readouterr().out


def test_without_headers_there_is_no_binding_and_no_error(monkeypatch, tmp_path, capsys):
    cpp_extension = pytest.importorskip("torch.utils.cpp_extension")
    monkeypatch.setattr(build, "STEP", str(tmp_path / "_step.so"))
    monkeypatch.setattr(cpp_extension, "include_paths", lambda *a, **k: [])
    build._binding()
    assert not os.listdir(tmp_path) and "python_variable.h" in capsys.readouterr().out


def test_a_binding_that_does_not_compile_is_an_error(monkeypatch, tmp_path):
    pytest.importorskip("torch")
    monkeypatch.setattr(build, "STEP", str(tmp_path / "_step.so"))

    def fails(cmd, **_):
        return subprocess.CompletedProcess(cmd, 1, "", "no such thing")
    monkeypatch.setattr(build.subprocess, "run", fails)
    monkeypatch.setattr(build.shutil, "which", lambda name: "/usr/bin/" + name)
    with pytest.raises(RuntimeError, match="no such thing"):
        build._binding()
