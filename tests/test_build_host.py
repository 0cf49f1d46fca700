"""The short way from torch tensors (bind/fastcall.cpp) is optional: neither its build nor its file can keep the CUDA library
from being built or used.  No GPU is touched."""
import subprocess

import pytest
import torch

from sonata_b200 import build
from sonata_b200.kernels import _common


@pytest.fixture
def common(monkeypatch):
    build.build()
    monkeypatch.setattr(_common, "_fast", None)
    return _common


def test_library_is_built_where_the_short_way_cannot_be(monkeypatch, tmp_path):
    """Without g++ (or torch's or Python's headers) build() still gives the library, and says what is missing."""
    run = subprocess.run

    def without_gxx(cmd, *a, **k):
        if cmd[0] == "g++":
            raise FileNotFoundError("g++")
        return run(cmd, *a, **k)
    bind = tmp_path / "bind.cpp"
    bind.write_text(build.BIND_SRC.read_text())  # newer than what is built
    monkeypatch.setattr(build, "BIND_SRC", bind)
    monkeypatch.setattr(build.subprocess, "run", without_gxx)
    with pytest.warns(UserWarning, match="g\\+\\+"):
        assert build.build() == build.LIB and build.LIB.exists()


@pytest.mark.parametrize("other", ["torch", "python", "abi"])
def test_another_interpreter_or_torch_has_another_file(monkeypatch, other):
    here = build.bind_path()
    if other == "torch":
        monkeypatch.setattr(torch, "__version__", "9.9.9")
    elif other == "python":
        monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-399")
    else:
        monkeypatch.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
    assert build.bind_path() != here


def test_a_file_that_does_not_load_is_left_out(common, monkeypatch, tmp_path):
    bad = tmp_path / "_fastcall.bad.so"
    bad.write_bytes(b"not a shared object")
    monkeypatch.setattr(build, "bind_path", lambda: bad)
    with pytest.warns(UserWarning, match="_fastcall.bad.so"):
        assert common.fast() is common._NoFast
    assert common.fast() is common._NoFast  # and says so once


def test_no_file(common, monkeypatch, tmp_path):
    monkeypatch.setattr(build, "bind_path", lambda: tmp_path / "none.so")
    assert common.fast() is common._NoFast


def test_the_file_that_was_built_loads(common):
    f = common.fast()
    assert f is not common._NoFast and f.attend() is None
