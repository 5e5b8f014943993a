"""CPU: when the torch extension is built again."""
import os
from pathlib import Path
from types import SimpleNamespace

import pytest

pytest.importorskip("torch")
from helix_b200 import build  # noqa: E402


def test_another_torch_builds_the_extension_again(monkeypatch, tmp_path):
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_bytes(b"")
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    version = ["2.11.0"]
    monkeypatch.setattr(build, "BUILD", tmp_path)
    monkeypatch.setattr(build, "TORCH_EXT", tmp_path / "ext.so")
    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr("importlib.metadata.version", lambda name: version[0])
    build._build_torch(False)
    assert len(ran) == 1
    build._build_torch(False)
    assert len(ran) == 1                       # nothing changed
    version[0] = "2.12.0"
    build._build_torch(False)
    assert len(ran) == 2                       # built against another torch
    build._build_torch(False)
    assert len(ran) == 2
    monkeypatch.setenv("CXX", "another-compiler")
    build._build_torch(False)
    assert len(ran) == 3 and ran[-1][0] == "another-compiler"
    os.utime(build.TORCH_EXT, (0, 0))          # older than its source
    build._build_torch(False)
    assert len(ran) == 4
    build._build_torch(True)
    assert len(ran) == 5
