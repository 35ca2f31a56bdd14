"""What build.py compiles and when, with a compiler that only notes its command lines."""
import importlib
import os

import pytest

from gemma_npu_b200 import build


@pytest.fixture
def compiler(tmp_path, monkeypatch):
    """An empty source tree with the binding's source; the commands run, whose outputs are made empty."""
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "decode_binding.cpp").write_text("")
    (tmp_path / "include").mkdir()
    for name, at in (("CSRC", "csrc"), ("INCLUDE", "include"), ("BUILD", "_build"), ("LIB", "lib.so"), ("BINDING", "_decode.so")):
        monkeypatch.setattr(build, name, str(tmp_path / at))
    commands = []

    def run(cmd, check):
        commands.append(os.path.basename(cmd[0]))
        open(cmd[cmd.index("-o") + 1], "w").close()

    monkeypatch.setattr(build, "nvcc_path", lambda: "/cuda/bin/nvcc")
    monkeypatch.setattr(build.subprocess, "run", run)
    return commands


def test_both_are_built_once(compiler):
    assert build.build(quiet=True) == build.LIB
    assert compiler == ["nvcc", "g++"] and os.path.exists(build.BINDING)
    build.build(quiet=True)
    assert compiler == ["nvcc", "g++"]


def test_without_torch_the_library_is_built(compiler, monkeypatch, capsys):
    """A C caller has nvcc and no torch."""
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setitem(build.sys.modules, "torch", None)  # (importing it raises ImportError)
    assert build.build() == build.LIB and os.path.exists(build.LIB)
    assert compiler == ["nvcc"] and not os.path.exists(build.BINDING)
    assert "no torch" in capsys.readouterr().out


def test_the_binding_is_built_anew_for_another_torch_or_python(compiler, monkeypatch):
    import sysconfig

    import torch

    build.build_binding(quiet=True)
    assert compiler == ["g++"]
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build.build_binding(quiet=True)
    assert compiler == ["g++"] * 2
    build.build_binding(quiet=True)
    assert compiler == ["g++"] * 2
    monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "another")
    build.build_binding(quiet=True)
    assert compiler == ["g++"] * 3
