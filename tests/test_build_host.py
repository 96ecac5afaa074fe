"""CPU: when the tensor-level module is built, built again and left out."""
import os
import time

import pytest

from hybrid_llm_b200 import _native, build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """The module's build in a folder of its own, its compiler a recorder."""
    monkeypatch.setattr(build, "TORCH_LIB", tmp_path / "llmyb_torch.so")
    monkeypatch.setattr(build, "BUILD", tmp_path)
    made = []

    def compiled(verbose):
        made.append(1)
        build.TORCH_LIB.write_text("module")
    monkeypatch.setattr(build, "_torch_module", compiled)
    return made


def test_built_once_and_again_when_an_input_changes(tree, monkeypatch):
    build._build_torch_module(False, False)
    build._build_torch_module(False, False)
    assert len(tree) == 1
    build._build_torch_module(True, False)
    assert len(tree) == 2
    monkeypatch.setattr(build.importlib.metadata, "version", lambda name: "0.0.1")
    build._build_torch_module(False, False)
    build._build_torch_module(False, False)
    assert len(tree) == 3                       # another torch
    old = time.time() - 10 ** 9
    os.utime(build.TORCH_LIB, (old, old))
    build._build_torch_module(False, False)
    assert len(tree) == 4                       # newer sources


@pytest.mark.parametrize("gone", ["torch", "g++"])
def test_left_out_where_its_needs_are_missing(tree, monkeypatch, capsys, gone):
    """The native library is built without it; an older module does not stay behind."""
    build.TORCH_LIB.write_text("of older sources")
    if gone == "torch":
        monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    else:
        monkeypatch.setattr(build.shutil, "which", lambda name: None)
    build._build_torch_module(False, False)
    assert not tree and not build.TORCH_LIB.exists() and gone in capsys.readouterr().err


def test_absent_module_raises(tmp_path, monkeypatch):
    monkeypatch.setattr(_native, "_torch_module", None)
    monkeypatch.setattr(_native, "TORCH_LIB_PATH", tmp_path / "llmyb_torch.so")
    with pytest.raises(RuntimeError, match="torch module not found"):
        _native.torch_module()
