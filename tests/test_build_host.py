"""When the Python binding is built again: its torch and Python have to be those it was
compiled against, and the C library alone needs neither."""
import importlib.metadata
import importlib.util
import os
import subprocess
from pathlib import Path

import pytest

spec = importlib.util.spec_from_file_location(
    "qcau_build", Path(__file__).resolve().parent.parent / "deepseek-v4-flash_b200" / "build.py")
B = importlib.util.module_from_spec(spec)
spec.loader.exec_module(B)


@pytest.fixture
def compiler(tmp_path, monkeypatch):
    """The calls of the compiler, which writes an empty file here."""
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_bytes(b"")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(B.subprocess, "run", run)
    monkeypatch.setattr(B, "BIND", tmp_path / "_bind.so")
    monkeypatch.setattr(B, "BIND_STAMP", tmp_path / "build" / "bind.stamp")
    return calls


def test_binding_is_built_once_for_a_torch(compiler, monkeypatch):
    B.build_bind()
    assert len(compiler) == 1
    B.build_bind()
    assert len(compiler) == 1
    B.build_bind(force=True)
    assert len(compiler) == 2
    version = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: version(name) + ".later")
    B.build_bind()
    B.build_bind()
    assert len(compiler) == 3


def test_binding_of_another_python_or_of_unknown_origin_is_built_again(compiler, monkeypatch):
    B.build_bind()
    B.BIND_STAMP.unlink()
    B.build_bind()
    assert len(compiler) == 2
    monkeypatch.setattr(B.sysconfig, "get_config_var", lambda name: "cpython-399")
    B.build_bind()
    assert len(compiler) == 3


def test_binding_follows_its_source(compiler):
    B.build_bind()
    os.utime(B.BIND, (1, 1))
    B.build_bind()
    assert len(compiler) == 2


def test_library_alone_without_torch(compiler, monkeypatch, capsys):
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: None)
    B.build_bind()
    assert not compiler and "without its Python binding" in capsys.readouterr().err
