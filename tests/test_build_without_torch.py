"""CPU: the C library is built whatever becomes of its torch binding (no compiler runs here)."""

from __future__ import annotations

import importlib.util
import subprocess
from pathlib import Path

import pytest

from axiom_amd import build as B


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """build() with its outputs in tmp_path and compilers that only write their output file."""
    def run(cmd, **kw):
        cmd = [str(c) for c in cmd]
        if tree.fail and any(tree.fail in c for c in cmd):
            return subprocess.CompletedProcess(cmd, 1, "", "no such header")
        Path(cmd[cmd.index("-o") + 1]).write_text("built")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    class tree:   # noqa: N801
        fail = None
        lib, binding = tmp_path / "libkda_mi355x.so", tmp_path / "_latent_torch.so"
    monkeypatch.setattr(B, "LIB", tree.lib)
    monkeypatch.setattr(B, "BINDING", tree.binding)
    monkeypatch.setattr(B, "BUILD", tmp_path / "_build")
    monkeypatch.setattr(B, "_hipcc", lambda: "hipcc")
    monkeypatch.setattr(B.subprocess, "run", run)
    return tree


def test_all(tree):
    assert B.build() == tree.lib and tree.lib.exists() and tree.binding.exists()


def test_binding_that_does_not_compile(tree):
    tree.fail = "latent_torch.cpp"
    with pytest.raises(RuntimeError, match="latent_torch.cpp"):
        B.build()
    assert tree.lib.exists() and not tree.binding.exists()


def test_no_torch(tree, monkeypatch, capsys):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setitem(__import__("sys").modules, "torch", None)   # importing it raises
    assert B.build() == tree.lib and tree.lib.exists() and not tree.binding.exists()
    assert "_latent_torch.so" in capsys.readouterr().err


def test_library_that_does_not_compile(tree):
    tree.fail = "kda_chunk.hip"
    with pytest.raises(RuntimeError, match="kda_chunk.hip"):
        B.build()
    assert not tree.lib.exists()
