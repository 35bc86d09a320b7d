"""When the libraries are built again (CPU; nothing is compiled)."""

from __future__ import annotations

import os

import pytest
import torch

from ataraxos_b200 import build as B


@pytest.fixture
def built(tmp_path, monkeypatch):
    """A build directory with every library up to date; the names of those that a build() makes again."""
    made = []
    for name in ("LIB_PATH", "DEBUG_LIB_PATH", "TORCH_LIB_PATH", "TORCH_STAMP"):
        monkeypatch.setattr(B, name, tmp_path / getattr(B, name).name)
        getattr(B, name).write_text("")
    B.TORCH_STAMP.write_text(B._torch_in_use())
    monkeypatch.setattr(B, "LIB_DIR", tmp_path)
    monkeypatch.setattr(B, "_compile", lambda path, extra, verbose: made.append(path.name))
    monkeypatch.setattr(B, "_compile_torch", lambda verbose: made.append(B.TORCH_LIB_PATH.name))
    return made


def test_nothing_is_built_twice(built):
    B.build()
    assert built == []


def test_another_torch_builds_the_torch_operators_again(built, monkeypatch):
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    B.build()
    assert built == [B.TORCH_LIB_PATH.name]


@pytest.mark.parametrize("lost", ["TORCH_STAMP", "TORCH_LIB_PATH"])
def test_an_unknown_torch_builds_the_torch_operators_again(built, lost):
    getattr(B, lost).unlink()
    B.build()
    assert built == [B.TORCH_LIB_PATH.name]


def test_older_than_its_source_is_built_again(built):
    os.utime(B.TORCH_LIB_PATH, (1, 1))
    B.build()
    assert built == [B.TORCH_LIB_PATH.name]
