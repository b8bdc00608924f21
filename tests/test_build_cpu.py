"""The library is built whether or not the module that packs torch tensors can be."""
import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest

from g4b_b200 import build


@pytest.fixture
def fake(monkeypatch, tmp_path):
    """build() in a folder of its own, with compilers that only write their output files."""
    state = SimpleNamespace(commands=[], gxx=0, dir=tmp_path)
    for name, file in (("LIBDIR", ""), ("LIB", "libg4b_attn.so"), ("VIEWS", "_views.so")):
        monkeypatch.setattr(build, name, tmp_path / file if file else tmp_path)

    def run(cmd, **kw):
        state.commands.append(Path(cmd[0]).name)
        if cmd[0] == "g++":
            if state.gxx is None:
                raise FileNotFoundError("g++")
            if state.gxx:
                return SimpleNamespace(returncode=state.gxx, stdout="", stderr="c10/cuda/CUDAStream.h: no such file")
        Path(cmd[cmd.index("-o") + 1]).write_text("x")
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    return state


def test_both_are_built_once(fake):
    build.build()
    assert build.LIB.exists() and build.VIEWS.exists() and fake.commands.count("g++") == 1
    n = len(fake.commands)
    build.build()
    assert len(fake.commands) == n
    build.VIEWS.unlink()
    build.build()
    assert build.VIEWS.exists()


@pytest.mark.parametrize("why", [1, None])
def test_the_library_is_built_without_the_module(fake, why, capfd):
    build.VIEWS.write_text("of another torch")
    fake.gxx = why
    assert build.build() == build.LIB and build.LIB.exists() and not build.VIEWS.exists()
    assert "packing stays in Python" in capfd.readouterr().err
    n = len(fake.commands)
    build.build()                                   # nothing changed: not tried again
    assert len(fake.commands) == n
    fake.gxx = 0
    build.build(force=True)
    assert build.VIEWS.exists()


def test_the_library_is_built_without_headers_or_torch(fake, monkeypatch):
    import torch.utils.cpp_extension as cpp

    def none(*a, **kw):
        raise RuntimeError("no CUDA in this torch")

    monkeypatch.setattr(cpp, "include_paths", none)
    build.build()
    assert build.LIB.exists() and not build.VIEWS.exists()
    monkeypatch.setattr(build, "_torch_version", lambda: "")
    build.VIEWS.write_text("of a torch that is gone")
    build.build()
    assert build.LIB.exists() and not build.VIEWS.exists()


def test_a_broken_kernel_still_fails(fake, monkeypatch):
    run = subprocess.run
    monkeypatch.setattr(subprocess, "run", lambda cmd, **kw: SimpleNamespace(returncode=1, stdout="", stderr="error") if "nvcc" in cmd[0] else run(cmd, **kw))
    with pytest.raises(RuntimeError, match="nvcc failed"):
        build.build()


def test_another_interpreter_is_another_build(monkeypatch):
    one = build._digest()
    monkeypatch.setattr(sys, "version", "3.99.0 (another)")
    assert build._digest() != one
