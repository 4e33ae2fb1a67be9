"""The in-tree build where torch is missing or another one than the binding was built against."""
import os
import subprocess
import types

import pytest

from rocwmma_b200 import build as B


@pytest.mark.parametrize("cpu_only", [False, True])
def test_the_c_libraries_are_built_without_torch(monkeypatch, tmp_path, cpu_only):
    linked = []
    spec = types.SimpleNamespace(origin=str(tmp_path / "torch" / "__init__.py")) if cpu_only else None
    monkeypatch.setattr(B.importlib.util, "find_spec", lambda name: spec)
    monkeypatch.setattr(B, "_stale", lambda target, sources: target.endswith("_bind.so"))
    monkeypatch.setattr(B, "_link", lambda objs, name, force: linked.append(name) or name)
    assert B.build() == ("libb200wmma.so", "libb200wmma_test.so")
    assert linked == ["libb200wmma.so", "libb200wmma_test.so"]


@pytest.fixture
def built(monkeypatch, tmp_path):
    """A binding that is newer than its sources, and the compiler calls that _bind() makes."""
    calls = []
    monkeypatch.setattr(B, "HERE", str(tmp_path))
    monkeypatch.setattr(B, "LIB", str(tmp_path))
    (tmp_path / "_bind.so").write_bytes(b"")
    monkeypatch.setattr(B.subprocess, "run", lambda cmd, **_: calls.append(cmd) or subprocess.CompletedProcess(cmd, 0, "", ""))
    B._bind(False)
    return calls


def test_the_binding_is_built_again_for_another_torch(built, monkeypatch):
    before = len(built)
    assert B._bind(False) == os.path.join(B.HERE, "_bind.so") and len(built) == before
    monkeypatch.setattr(B.importlib.metadata, "version", lambda name: "99.0")
    B._bind(False)
    assert len(built) == before + 1
    B._bind(False)
    assert len(built) == before + 1


def test_a_binding_that_failed_to_build_is_tried_again(built, monkeypatch):
    monkeypatch.setattr(B.importlib.metadata, "version", lambda name: "99.0")
    monkeypatch.setattr(B.subprocess, "run", lambda cmd, **_: subprocess.CompletedProcess(cmd, 1, "", "no"))
    for _ in range(2):
        with pytest.raises(RuntimeError, match="bind.cpp"):
            B._bind(False)
