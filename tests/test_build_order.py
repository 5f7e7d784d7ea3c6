"""What a failing compile of the torch module leaves built (CPU only, nothing is compiled)."""

from __future__ import annotations

import subprocess
from types import SimpleNamespace

import pytest

from light_vllm_b200 import build


def test_the_library_does_not_wait_for_the_torch_module(monkeypatch, tmp_path):
    """Only the 8-bit cache's and the draft verification's calls go through the torch module: without it
    the library and the metadata module are built all the same, and the build still fails."""

    ran = []

    def no_torch(force=False):
        ran.append("torch")
        raise RuntimeError("csrc/torch_ops.cpp is compiled against torch, which is not installed")

    def run(cmd, **kwargs):
        ran.append("library")
        (tmp_path / "liblvb200.so.tmp").write_text("")
        return SimpleNamespace(returncode=0, stderr="")

    monkeypatch.setattr(build, "OUTPUT", tmp_path / "liblvb200.so")
    monkeypatch.setattr(build, "build_hostpack", lambda force=False: ran.append("metadata"))
    monkeypatch.setattr(build, "build_torch_ops", no_torch)
    monkeypatch.setattr(subprocess, "run", run)
    with pytest.raises(RuntimeError, match="torch_ops.cpp"):
        build.build()
    assert set(ran) == {"metadata", "library", "torch"} and (tmp_path / "liblvb200.so").is_file()
    ran.clear()
    with pytest.raises(RuntimeError, match="torch_ops.cpp"):  # current now, and the module still missing
        build.build()
    assert "torch" in ran and "library" not in ran
