"""The library without csrc/calls.cpp: not built, built with another torch, no C++ compiler."""

import os
import subprocess
import sys

import pytest
import torch

import xb200
from xb200 import build, ops


@pytest.fixture
def unbound(monkeypatch):
    """ops before its first call."""
    real = ops._direct()
    with monkeypatch.context() as m:
        m.setattr(ops, "_calls", None)
        yield m
    assert ops._direct() is real


def _left_alone():
    with pytest.warns(RuntimeWarning, match="_calls.so is not used"):
        direct = ops._direct()
    assert ops._direct() is direct  # and says it once
    x = torch.zeros((2, 3))
    assert direct.beam_select(x, x, 2) is None
    assert direct.paged_attention(*[x] * 7, 0.5, None, None) is False
    assert direct.paged_rope_kv(x, None, None, *[x] * 6, None, None) is False
    assert direct.paged_read_kv(*[x] * 7, None, None) is False
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_select(x, x, 2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(*[x] * 7, 0.5)


def test_not_built(unbound):
    unbound.delattr(xb200, "_calls", raising=False)
    unbound.setitem(sys.modules, "xb200._calls", None)  # what the import finds where there is no such file
    _left_alone()


def test_built_with_another_torch(unbound):
    from xb200 import _calls

    assert _calls.torch_version == torch.__version__
    unbound.setattr(_calls, "torch_version", "1.0")
    _left_alone()


@pytest.mark.parametrize("fails", [lambda *a, **kw: subprocess.CompletedProcess(a, 1, "", "no headers"),
                                   lambda *a, **kw: (_ for _ in ()).throw(FileNotFoundError("g++"))])
def test_no_compiler(fails, tmp_path, monkeypatch):
    old = tmp_path / "_calls.so"
    old.write_bytes(b"an older one")
    os.utime(old, (0, 0))
    monkeypatch.setattr(build, "CALLS_PATH", str(old))
    monkeypatch.setattr(build.subprocess, "run", fails)
    with pytest.raises(RuntimeError, match="calls.cpp"):
        build.build_calls()
    assert not old.exists()


def test_the_library_is_built_without(monkeypatch):
    def fails():
        raise RuntimeError("g++ failed on calls.cpp")

    monkeypatch.setattr(build, "build_calls", fails)
    monkeypatch.setattr(build, "_compile", lambda src, extra: build.LIB_PATH)  # all of it is there
    with pytest.warns(RuntimeWarning, match="does without"):
        assert build.build() == build.LIB_PATH
