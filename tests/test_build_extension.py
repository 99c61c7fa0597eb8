"""build.py on hosts that differ from this one: without torch, with a torch that has no CUDA, with nvcc on the PATH
alone, and after a change of torch. No compiler is run."""
import importlib.util
import os
import sys

import pytest
import torch
from conftest import PKG_ROOT


@pytest.fixture
def build(monkeypatch, tmp_path):
    spec = importlib.util.spec_from_file_location("uwc_build", os.path.join(PKG_ROOT, "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.commands = []

    def run(cmd):
        m.commands.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
    monkeypatch.setattr(m.subprocess, "check_call", run)
    monkeypatch.setattr(m, "up_to_date", lambda: True)
    monkeypatch.setattr(m, "EXT_OUT", str(tmp_path / "_paged.so"))
    monkeypatch.setattr(m, "EXT_STAMP", str(tmp_path / "b" / "stamp"))
    return m


def test_a_host_without_torch_gets_the_library(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)        # import torch: ImportError
    assert build.build() == build.OUT and build.commands == []
    assert "_paged.so is not built" in capsys.readouterr().err


def test_a_torch_without_cuda_does_too(build, monkeypatch, capsys):
    monkeypatch.setattr(torch.version, "cuda", None)
    assert build.build() == build.OUT and build.commands == []
    assert "_paged.so is not built" in capsys.readouterr().err


def test_nvcc_on_the_path_gives_its_headers(build, monkeypatch, tmp_path):
    cuda = tmp_path / "toolkit"
    (cuda / "bin").mkdir(parents=True)
    (cuda / "bin" / "nvcc").write_text("#!/bin/sh\n")
    (cuda / "bin" / "nvcc").chmod(0o755)
    (tmp_path / "links").mkdir()
    (tmp_path / "links" / "nvcc").symlink_to(cuda / "bin" / "nvcc")
    monkeypatch.setenv("CUDA_HOME", str(tmp_path / "none"))
    for d in (cuda / "bin", tmp_path / "links"):
        monkeypatch.setenv("PATH", f"{d}:/bin")
        build.build_extension(force=True)
        assert f"-isystem{cuda}/include" in build.commands[-1]
    assert not [a for a in build.commands[-1] if a == "-isysteminclude"]


def test_another_torch_is_a_reason_to_build(build, monkeypatch):
    build.build_extension()
    assert len(build.commands) == 1
    build.build_extension()
    assert len(build.commands) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build.build_extension()
    assert len(build.commands) == 2
    build.build_extension()
    assert len(build.commands) == 2
