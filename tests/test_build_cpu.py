"""The build without what only the compiled callers need: the library is all that counts."""

import importlib
import subprocess
import sys

import pytest
import torch

from shellsmith_b200 import _build, _torch


@pytest.fixture
def callers(monkeypatch, tmp_path):
    """Callers of an older build in a place of their own; the library is up to date."""
    path = tmp_path / "_fastpath.so"
    path.write_bytes(b"old")
    monkeypatch.setattr(_build, "FASTPATH", path)
    monkeypatch.setattr(_build, "_stale", lambda: False)
    _build.os.utime(path, (1, 1))
    return path


def test_without_a_compiler(callers, monkeypatch):
    def run(cmd, **kw):
        raise FileNotFoundError(2, "No such file or directory", cmd[0])
    monkeypatch.setattr(_build.subprocess, "run", run)
    with pytest.warns(UserWarning, match="g\\+\\+"):
        assert _build.build() == _build.LIBRARY
    assert not callers.exists()


def test_without_headers(callers, monkeypatch):
    monkeypatch.setattr(_build.subprocess, "run", lambda cmd, **kw: subprocess.CompletedProcess(
        cmd, 1, "", "fatal error: Python.h: No such file or directory"))
    with pytest.warns(UserWarning, match="Python.h"):
        assert _build.build() == _build.LIBRARY
    assert not callers.exists()


def test_without_torch(callers, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)
    with pytest.warns(UserWarning, match="torch"):
        assert _build.build() == _build.LIBRARY
    assert not callers.exists()


def test_up_to_date_callers_stay(callers, monkeypatch):
    callers.touch()
    monkeypatch.setattr(_build.subprocess, "run", lambda *a, **kw: pytest.fail("compiled"))
    assert _build.build() == _build.LIBRARY
    assert callers.read_bytes() == b"old"


def test_a_built_library_needs_no_toolkit(callers, monkeypatch):
    def missing():
        raise RuntimeError("nvcc not found")
    monkeypatch.setattr(_build, "nvcc", missing)
    with pytest.warns(UserWarning, match="nvcc not found"):
        assert _build.build() == _build.LIBRARY
    assert not callers.exists()


def test_callers_of_another_torch_are_not_used(monkeypatch):
    if _torch.fast is None:
        pytest.skip("the compiled callers are not built")
    assert _torch.fast.torch_version == torch.__version__
    try:
        with monkeypatch.context() as m:
            m.setattr(torch, "__version__", "0.0.1")
            assert importlib.reload(_torch).fast is None
    finally:
        assert importlib.reload(_torch).fast is not None
