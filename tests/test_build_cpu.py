"""The build script with its compilers replaced: what is built again when, and that the library does not depend on the module for torch."""
import importlib.util
import os
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "cpm.cu_b200")


@pytest.fixture()
def script(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("build_under_test", os.path.join(PKG, "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    monkeypatch.setattr(b, "OBJ_DIR", str(tmp_path / "build"))
    monkeypatch.setattr(b, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(b, "OPS", str(tmp_path / "ops.so"))
    b.ran, b.broken = [], set()

    def run(cmd, what):
        kind = "module" if cmd[0] == "g++" else "link" if "-shared" in cmd else "object"
        b.ran.append(kind)
        if kind in b.broken:
            raise RuntimeError(what)
        open(cmd[cmd.index("-o") + 1], "w").close()
    monkeypatch.setattr(b, "_run", run)
    return b


def kinds(b):
    got, b.ran = sorted(set(b.ran)), []
    return got


def test_library_and_module_are_built_once(script):
    assert script.build(verbose=False) == script.LIB and kinds(script) == ["link", "module", "object"]
    script.build(verbose=False)
    assert kinds(script) == []
    script.build(force=True, verbose=False)
    assert kinds(script) == ["link", "module", "object"]


def test_library_without_torch(script, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)          # importing it raises ImportError
    assert script.build(verbose=False) == script.LIB and kinds(script) == ["link", "object"]
    assert "no torch" in capsys.readouterr().out
    script.build(verbose=False)
    assert kinds(script) == []


def test_a_module_that_does_not_compile_leaves_the_library(script):
    script.broken = {"module"}
    for expected in (["link", "module", "object"], ["module"]):
        with pytest.raises(RuntimeError, match="torch_ops.cpp"):
            script.build(verbose=False)
        assert kinds(script) == expected
    script.broken = set()
    script.build(verbose=False)
    assert kinds(script) == ["module"]


def test_another_torch_needs_another_module(script, monkeypatch):
    import torch
    script.build(verbose=False)
    kinds(script)
    monkeypatch.setattr(torch, "__version__", "0.0")
    script.build(verbose=False)
    assert kinds(script) == ["module"]


def test_a_build_that_fails_does_not_count(script):
    script.build(verbose=False)
    script.broken = {"link"}
    with pytest.raises(RuntimeError):
        script.build(force=True, verbose=False)
    script.broken = set()
    kinds(script)
    script.build(verbose=False)
    assert kinds(script) == ["link", "object"]
