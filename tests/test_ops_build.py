"""When the torch binding of the operators is rebuilt, left out, and what is said where it is missing; on
the host, with a torch of a few files and a recorded compiler."""
from __future__ import annotations

import importlib.machinery
import os

import pytest

import z2b.build as B


@pytest.fixture
def made(tmp_path, monkeypatch):
    """A torch folder with CUDA's libraries, and the commands that build_ops runs instead of the compiler."""
    torch, ran = tmp_path / "torch", []
    (torch / "lib").mkdir(parents=True)
    (torch / "lib" / "libtorch_cuda.so").write_text("")
    (torch / "version.py").write_text("__version__ = '1'\n")
    spec = importlib.machinery.ModuleSpec("torch", None, is_package=True)
    spec.submodule_search_locations.append(str(torch))
    monkeypatch.setattr(B.importlib.util, "find_spec", lambda name: spec)
    monkeypatch.setattr(B, "BUILD", str(tmp_path / "_build"))
    monkeypatch.setattr(B, "OPS_LIB", str(tmp_path / "_ops.so"))

    def run(cmd):
        ran.append(cmd)
        open(B.OPS_LIB, "w").close()

    monkeypatch.setattr(B, "_run", run)
    return torch, ran


def test_the_binding_follows_torch(made):
    """Built once, again when torch or the interpreter is another, else not."""
    torch, ran = made
    assert B.build_ops() == B.OPS_LIB and len(ran) == 1
    assert B.build_ops() == B.OPS_LIB and len(ran) == 1
    (torch / "version.py").write_text("__version__ = '2'\n")
    B.build_ops()
    assert len(ran) == 2 and any(str(torch / "lib") in a for a in ran[-1])
    B.build_ops()
    os.remove(B.OPS_LIB)
    B.build_ops()
    assert len(ran) == 3


def test_a_build_that_failed_is_tried_again(made, monkeypatch):
    torch, ran = made
    B.build_ops()
    (torch / "version.py").write_text("__version__ = '2'\n")
    good = B._run

    def fails(cmd):
        raise RuntimeError("build failed")

    monkeypatch.setattr(B, "_run", fails)
    with pytest.raises(RuntimeError):
        B.build_ops()
    monkeypatch.setattr(B, "_run", good)
    B.build_ops()
    assert len(ran) == 2


def test_no_torch_with_cuda_no_binding(made, monkeypatch):
    """The rest of the library builds without torch, and beside one that has no CUDA."""
    torch, ran = made
    os.remove(torch / "lib" / "libtorch_cuda.so")
    assert B.build_ops() is None
    monkeypatch.setattr(B.importlib.util, "find_spec", lambda name: None)
    assert B.build_ops() is None and not ran


def test_a_missing_binding_says_what_to_do(monkeypatch):
    import importlib
    import sys

    pytest.importorskip("torch")
    import z2b
    import z2b.ops as was

    monkeypatch.setitem(sys.modules, "z2b._ops", None)       # an import of it fails
    monkeypatch.delattr(z2b, "_ops")
    monkeypatch.delitem(sys.modules, "z2b.ops")
    with pytest.raises(ImportError, match="build.py ops"):
        importlib.import_module("z2b.ops")
    monkeypatch.undo()
    assert importlib.import_module("z2b.ops") is was
