"""What the build compiles, and with what (no compiler runs)."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest

from gbxcule_amd import build


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """The commands of a build into an empty folder."""
    seen: list[list[str]] = []

    def run(batch, verbose):
        for cmd in batch:
            seen.append(cmd)
            Path(cmd[cmd.index("-o") + 1]).touch()

    monkeypatch.setattr(build, "_run", run)
    monkeypatch.setattr(build, "LIB_DIR", tmp_path)
    monkeypatch.setattr(build, "LIB_PATH", tmp_path / "libgbx_hip.so")
    monkeypatch.setattr(build, "EXT_PATH", tmp_path / "gbx_torch.so")
    return seen


def test_both_libraries(commands, tmp_path):
    assert build.build() == tmp_path / "libgbx_hip.so"
    assert {p.name for p in tmp_path.iterdir()} == {"libgbx_hip.so", "gbx_torch.so"}
    assert sum(str(build.CSRC / build.EXT_SOURCE) in c for c in commands) == 1
    for source in build.SOURCES:
        (cmd,) = [c for c in commands if str(build.CSRC / source) in c]
        assert "-packed-fp32-ops" in cmd and "--offload-arch=gfx950" in cmd


def test_without_torch_the_library_alone(commands, monkeypatch, tmp_path, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build() == tmp_path / "libgbx_hip.so"
    assert {p.name for p in tmp_path.iterdir()} == {"libgbx_hip.so"}
    assert "gbx_torch.so" in capsys.readouterr().err


def test_without_gcc_rocms_compiler(commands, monkeypatch, tmp_path):
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    build.build()
    (cmd,) = [c for c in commands if str(build.CSRC / build.EXT_SOURCE) in c]
    assert Path(cmd[0]).name == "amdclang++" and Path(cmd[0]).exists()
    assert (tmp_path / "gbx_torch.so").exists()
