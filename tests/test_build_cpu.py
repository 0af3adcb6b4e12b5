"""What is built when: the kernel library needs neither torch nor g++, the torch operators belong to one torch."""
import os
import types

import pytest

from ads_model_kernel_library_b200 import build as B


@pytest.fixture
def compiler(monkeypatch, tmp_path):
    """The build of this package with its outputs elsewhere and no source of the kernel library to compile; the commands that it runs."""
    commands = []

    def run(cmd, **how):
        commands.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(B.subprocess, "run", run)
    monkeypatch.setattr(B, "_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(B, "_sources", lambda: [])
    monkeypatch.setattr(B, "OUT", str(tmp_path / "kernels.so"))
    monkeypatch.setattr(B, "TORCH_OUT", str(tmp_path / "operators.so"))
    monkeypatch.setattr(B, "TORCH_STAMP", str(tmp_path / "build" / "stamp"), raising=False)
    return commands


def built(commands):
    return [os.path.basename(c[c.index("-o") + 1]) for c in commands]


def test_both_are_built_once(compiler):
    B.build()
    assert built(compiler) == ["kernels.so", "operators.so"]
    B.build()
    assert len(compiler) == 2
    B.build(force=True)
    assert len(compiler) == 4


@pytest.mark.parametrize("missing", ["torch", "g++"])
def test_without_torch_or_a_host_compiler(compiler, monkeypatch, missing, capsys):
    if missing == "torch":
        monkeypatch.setattr(B.importlib.util, "find_spec", lambda name: None)
    else:
        monkeypatch.setattr(B.shutil, "which", lambda name: None)
    assert B.build() == B.OUT
    assert built(compiler) == ["kernels.so"] and f"{missing} is not there" in capsys.readouterr().err


def test_another_torch(compiler, monkeypatch):
    B.build()
    version = B.importlib.metadata.version("torch")
    monkeypatch.setattr(B.importlib.metadata, "version", lambda name: version + ".post1")
    B.build()
    assert built(compiler) == ["kernels.so", "operators.so", "operators.so"]
    B.build()
    assert len(compiler) == 3
