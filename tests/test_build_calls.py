"""The library does without _calls.so: where PyTorch, its headers or a host compiler are missing the build leaves it out, and
the entry points go through ctypes then."""
import sys

import pytest
import torch

from amos_amd import build, ops


@pytest.mark.parametrize("missing", ["torch", "headers", "compiler"])
def test_build_leaves_the_calls_out(monkeypatch, tmp_path, capsys, missing):
    old = tmp_path / "_calls.so"
    old.write_bytes(b"of another PyTorch")
    monkeypatch.setattr(build, "CALLS", str(old))
    monkeypatch.setattr(build.subprocess, "check_call", lambda cmd: pytest.fail("compiled"))
    if missing == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    elif missing == "headers":
        monkeypatch.setattr(torch, "__file__", str(tmp_path / "__init__.py"))
    else:
        monkeypatch.setenv("CXX", "no-such-compiler -O1")
    assert build.build_calls(verbose=False) is None
    assert not old.exists() and "ctypes" in capsys.readouterr().out


def test_entry_points_without_the_calls(monkeypatch, tmp_path):
    monkeypatch.setattr(ops, "_CALLS_PATH", str(tmp_path / "_calls.so"))
    native = ops._Native()
    assert [getattr(native, name)(1, 2, 3) for name in ops._Native.NAMES] == [None] * len(ops._Native.NAMES)
    monkeypatch.setattr(ops, "_native", ops._Native())
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.group_norm(torch.zeros(1, 2, 2, 8), 2)


def test_calls_that_do_not_load_are_an_error(monkeypatch):
    monkeypatch.setattr(ops, "_CALLS_PATH", __file__)
    monkeypatch.setitem(sys.modules, "amos_amd._calls", None)
    monkeypatch.delattr(sys.modules["amos_amd"], "_calls", raising=False)
    with pytest.raises(RuntimeError, match="does not fit this PyTorch"):
        ops._Native().rows
