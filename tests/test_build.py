"""The build in a folder of its own: the library links whatever becomes of the
host extension, and the extension is rebuilt when what it was built for changes."""

import os
import subprocess
import sys

import pytest

from comfyui_vc_attention_b200 import build as B


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Two sources, and compilers that write the name of what they made."""
    src = tmp_path / "csrc"
    src.mkdir()
    (tmp_path / "include").mkdir()
    (tmp_path / "include" / "vcattn.h").write_text("")
    for name in ("one.cu", "two.cu", "host_ops.cpp"):
        (src / name).write_text("")
    for key, value in dict(CSRC=src, INCLUDE=tmp_path / "include", BUILD=tmp_path / "_build",
                           LIB=tmp_path / "lib.so", HOST_OPS=tmp_path / "_host_ops.so").items():
        monkeypatch.setattr(B, key, str(value))
    made, fails = [], set()

    def run(cmd, **_):
        out = cmd[cmd.index("-o") + 1]
        name = os.path.basename(out)
        made.append(name)
        if name in fails:
            return subprocess.CompletedProcess(cmd, 1, "", "no")
        with open(out, "w") as f:
            f.write(name)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(B.subprocess, "run", run)
    monkeypatch.setattr(B, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    return tmp_path, made, fails


def test_everything_once(tree):
    _, made, _ = tree
    B.build()
    assert sorted(made) == ["_host_ops.so.tmp", "lib.so.tmp", "one.o", "two.o"]
    made.clear()
    B.build()
    assert made == []


def test_without_torch_the_library_is_built(tree, monkeypatch, capsys):
    path, made, _ = tree
    monkeypatch.setitem(sys.modules, "torch", None)
    assert os.path.exists(B.build())
    assert sorted(made) == ["lib.so.tmp", "one.o", "two.o"] and not (path / "_host_ops.so").exists()
    assert "torch" in capsys.readouterr().err


def test_a_failing_extension_is_loud_and_leaves_a_linked_library(tree):
    path, made, fails = tree
    fails.add("_host_ops.so.tmp")
    with pytest.raises(RuntimeError, match="host_ops"):
        B.build()
    assert (path / "lib.so").exists()


def test_objects_newer_than_the_library_are_linked(tree):
    """As a build leaves them that compiled and then failed."""
    path, made, fails = tree
    B.build()
    later = os.path.getmtime(path / "lib.so") + 10
    os.utime(path / "_build" / "one.o", (later, later))
    made.clear()
    B.build()
    assert made == ["lib.so.tmp"]


def test_another_torch_rebuilds_the_extension(tree, monkeypatch):
    import torch
    _, made, _ = tree
    B.build()
    made.clear()
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    B.build()
    assert made == ["_host_ops.so.tmp"]
