"""Building the optional torch binding: the library's build succeeds without
it, and it is compiled again whenever what it was compiled from changes."""

import os
import subprocess
import sys
import time
import types
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def build(monkeypatch, tmp_path):
    """rns8_b200.build on a finished library in a folder of its own, with a
    compiler that records its commands and leaves a file."""
    from rns8_b200 import build

    include = tmp_path / "include"
    (include / "rns8").mkdir(parents=True)
    for name in ("rns8_quant.h", "abi.h", "status.h"):
        (include / "rns8" / name).write_text("")
    source = tmp_path / "quant_torch.cpp"
    source.write_text("")
    for name, value in dict(BUILD=tmp_path, LIB=tmp_path / "librns8.so", TORCH_LIB=tmp_path / "_quant_torch.so",
                            TORCH_SRC=source, INCLUDE=include).items():
        monkeypatch.setattr(build, name, value)
    monkeypatch.setattr(build, "sources", lambda: [])
    build.LIB.write_text("")
    build.runs, build.fails = [], False

    def run(cmd, **_):
        build.runs.append(cmd)
        if build.fails:
            return subprocess.CompletedProcess(cmd, 1, "", "no such header")
        Path(cmd[cmd.index("-o") + 1]).write_text("")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    yield build
    del build.runs, build.fails


def test_a_binding_that_does_not_compile_fails_itself_alone(build, capsys):
    build.TORCH_LIB.write_text("")  # of an earlier build
    build.fails = True
    assert build.build() == build.LIB
    assert "no such header" in capsys.readouterr().err
    assert not build.TORCH_LIB.exists()
    with pytest.raises(RuntimeError, match="no such header"):
        build.build_torch_binding()


@pytest.mark.parametrize("cuda,present", [(None, True), ("12.8", False)])
def test_no_binding_without_cuda_torch_or_python_headers(build, monkeypatch, tmp_path, cuda, present):
    fake = types.ModuleType("torch")
    fake.__dict__.update(__file__=str(tmp_path / "torch" / "__init__.py"), __version__="0",
                         version=types.SimpleNamespace(cuda=cuda),
                         _C=types.SimpleNamespace(_GLIBCXX_USE_CXX11_ABI=True))
    fake.__spec__ = torch.__spec__
    monkeypatch.setitem(sys.modules, "torch", fake)
    if not present:
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path / "nowhere")})
    assert build.build() == build.LIB and build.build_torch_binding(force=True) is None
    assert not build.runs


@pytest.mark.parametrize("name", ["rns8_quant.h", "abi.h", "status.h"])
def test_compiled_again_when_a_header_changes(build, name):
    assert build.build_torch_binding() == build.TORCH_LIB and len(build.runs) == 1
    assert build.build_torch_binding() == build.TORCH_LIB and len(build.runs) == 1
    later = time.time() + 10
    os.utime(build.INCLUDE / "rns8" / name, (later, later))
    build.build_torch_binding()
    assert len(build.runs) == 2


def test_compiled_again_when_the_command_changes(build, monkeypatch):
    build.build_torch_binding()
    paths = build.sysconfig.get_paths()
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {**paths, "include": paths["include"] + "/."})
    build.build_torch_binding()
    assert len(build.runs) == 2


def test_warnings_of_the_bindings_own_code_are_shown(build, monkeypatch, capsys):
    run = build.subprocess.run

    def warn(cmd, **kwargs):
        run(cmd, **kwargs)
        return subprocess.CompletedProcess(cmd, 0, "", "quant_torch.cpp: warning: unused variable")

    monkeypatch.setattr(build.subprocess, "run", warn)
    build.build_torch_binding()
    cmd = build.runs[0]
    assert "-w" not in cmd and "-Wall" in cmd and f"-I{build.INCLUDE}" in cmd
    assert all(not c.startswith("-I") or c == f"-I{build.INCLUDE}" for c in cmd)  # the rest are system headers
    assert "unused variable" in capsys.readouterr().err
