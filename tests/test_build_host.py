"""What the build keeps apart: bindings of other torch or Python versions, processes that build at once, and the
library where there is no torch.  The compilers are stand-ins."""

import os
import subprocess
import sysconfig
from pathlib import Path

import pytest
import torch

import rldx_b200  # noqa: F401
from rldx_b200 import _lib, build


@pytest.fixture
def compilers(monkeypatch, tmp_path):
    """The build in an empty folder, with compilers that write their output's name into it."""
    runs = []

    def run(cmd, **kw):
        out = Path(cmd[cmd.index("-o") + 1])
        runs.append(out)
        out.write_text(out.name)
        return subprocess.CompletedProcess(cmd, 1 if "fail" in os.environ.get("CXX", "") else 0, "", "what it says")

    monkeypatch.setattr(build, "PKG_DIR", tmp_path)
    monkeypatch.setattr(build, "LIB_PATH", tmp_path / build.LIB_NAME)
    monkeypatch.setattr(subprocess, "run", run)
    return runs


def test_the_loaded_binding_is_this_torchs(lib):
    mod = _lib.load_binding()
    assert Path(mod.__file__) == build.binding_path() and not build.binding_needs_build()
    assert torch.__version__ in build.binding_path().name and sysconfig.get_config_var("SOABI") in build.binding_path().name


def test_another_torch_gets_a_binding_of_its_own(compilers, monkeypatch, tmp_path):
    first = build.build_binding()
    assert first.exists() and not build.binding_needs_build()
    monkeypatch.setattr(build, "torch_version", lambda: "9.9.0+cu1")
    assert build.binding_needs_build()
    second = build.build_binding()
    assert second != first and first.exists() and second.exists() and len(compilers) == 2
    monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "cpython-399-other")
    assert build.binding_needs_build() and build.binding_path() not in (first, second)


def test_the_library_is_built_without_torch(compilers, monkeypatch, tmp_path):
    monkeypatch.setattr(build, "torch_version", lambda: None)
    assert build.build() == tmp_path / build.LIB_NAME
    assert [p.name for p in tmp_path.iterdir()] == [build.LIB_NAME] and len(compilers) == 1


def test_processes_do_not_share_their_output(compilers, monkeypatch, tmp_path):
    build.build()
    assert len(compilers) == 2 and all(f".{os.getpid()}." in p.name for p in compilers)
    monkeypatch.setattr(os, "getpid", lambda: 7)
    build.build(force=True)
    assert len(set(compilers)) == 4
    assert sorted(p.name for p in tmp_path.iterdir()) == sorted([build.LIB_NAME, build.binding_path().name])


def test_a_failed_build_leaves_what_was_there(compilers, monkeypatch, tmp_path):
    path = build.build_binding()
    before = path.read_text()
    monkeypatch.setenv("CXX", "fail")
    with pytest.raises(RuntimeError, match="fail failed"):
        build.build_binding(force=True)
    assert path.read_text() == before and [p.name for p in tmp_path.iterdir()] == [path.name]
