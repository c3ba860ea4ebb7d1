"""__graft_entry__: what build() compiles and when, and what smoke() notices about the libraries that it runs."""
import os
import subprocess

import pytest

import __graft_entry__ as entry


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Libraries newer than their sources, in a folder of their own; the commands that build() would run are recorded instead."""
    sources = {}
    for out, deps in (("lib.so", ("a.hip", "b.hip")), ("host.so", ("h.cpp",)), ("ext.so", ("t.cpp",))):
        for name in deps + (out,):
            (tmp_path / name).write_text("")
            os.utime(tmp_path / name, (2000, 2000) if name == out else (1000, 1000))
        sources[str(tmp_path / out)] = [str(tmp_path / d) for d in deps]
    for name, out in zip(("LIB", "HOST_LIB", "EXT_LIB"), sources):
        monkeypatch.setattr(entry, name, out)
    monkeypatch.setattr(entry, "_sources", lambda: sources)
    monkeypatch.setattr(entry, "_units", lambda: sources[entry.LIB])
    built = []

    class Popen:
        def __init__(self, cmd):
            built.append(cmd[-1])
            self.returncode = 0

        def wait(self):
            return 0
    monkeypatch.setattr(subprocess, "Popen", Popen)
    monkeypatch.setattr(subprocess, "check_call", lambda cmd: built.append(next(c for c in cmd if c.endswith(".so"))))
    import ctypes
    import types
    from gnn_model_explainer_amd import engine
    monkeypatch.setattr(ctypes, "CDLL", lambda path: None)
    monkeypatch.setattr(engine, "bind", lambda lib: types.SimpleNamespace(gnnx_version=lambda: b""))
    return types.SimpleNamespace(path=tmp_path, built=lambda: [os.path.basename(b) for b in built if b.endswith(".so")], clear=built.clear)


def test_build_compiles_everything_unless_told_otherwise(tree, monkeypatch):
    """... also inside a test: what decides is an argument or an environment variable of its own, not the test runner's."""
    assert "PYTEST_CURRENT_TEST" in os.environ
    monkeypatch.delenv("GNNX_BUILD_STALE_ONLY")
    entry.build()
    assert tree.built() == ["lib.so", "host.so", "ext.so"]
    tree.clear()
    entry.build(stale_only=True)
    assert tree.built() == []
    monkeypatch.setenv("GNNX_BUILD_STALE_ONLY", "1")
    entry.build()
    assert tree.built() == []
    os.utime(tree.path / "b.hip", (3000, 3000))
    (tree.path / "ext.so").unlink()
    entry.build()
    assert tree.built() == ["lib.so", "ext.so"]
    tree.clear()
    entry.build(stale_only=False)
    assert tree.built() == ["lib.so", "host.so", "ext.so"]


def test_smoke_says_which_libraries_are_older_than_their_sources_and_builds_missing_ones(tree, monkeypatch, capsys):
    import torch
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    with pytest.raises(AssertionError, match="cuda:0"):
        entry.smoke()
    assert tree.built() == [] and "OLDER" not in capsys.readouterr().err
    os.utime(tree.path / "t.cpp", (3000, 3000))
    with pytest.raises(AssertionError, match="cuda:0"):
        entry.smoke()
    err = capsys.readouterr().err
    assert "ext.so is OLDER THAN ITS SOURCES" in err and "lib.so" not in err and tree.built() == []
    (tree.path / "host.so").unlink()
    with pytest.raises(AssertionError, match="cuda:0"):
        entry.smoke()
    assert tree.built() == ["host.so", "ext.so"]


def test_the_sources_are_the_trees(monkeypatch):
    src = entry._sources()
    assert all(os.path.exists(s) for deps in src.values() for s in deps)
    names = {os.path.basename(s) for s in src[entry.LIB]}
    assert {"gnnx_capi.hip", "gnnx_ops.hip", "gnnx_norm.hpp", "gnnx_error.hpp", "gnnx.h"} <= names
