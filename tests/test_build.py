"""The build without a compiler: what is compiled, linked and rebuilt, and what a failure leaves behind."""
import os
import subprocess
import sys
from types import SimpleNamespace

import pytest

from cubutterfly_b200 import _build


@pytest.fixture
def build(tmp_path, monkeypatch):
    """build() over one unit in a folder of its own; `ran` lists what was made, `failing` holds what fails."""
    obj = tmp_path / "obj" / "unit.o"
    paths = dict(OBJ=obj.parent, LIB_DIR=tmp_path / "lib", LIB=tmp_path / "lib" / "lib.so",
                 TORCH_EXT=tmp_path / "ext.so")
    for name, path in paths.items():
        monkeypatch.setattr(_build, name, path)
    monkeypatch.setattr(_build, "_units", lambda: [(["cc", "-o", str(obj)], _build.CSRC / "unit.cu", obj)])
    ran, failing = [], set()

    def run(cmd, **kwargs):
        target = cmd[cmd.index("-o") + 1]
        ran.append(os.path.basename(target))
        if ran[-1] in failing:
            return subprocess.CompletedProcess(cmd, 1, "", "it failed")
        open(target, "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(_build.subprocess, "run", run)

    def call():
        ran.clear()
        return _build.build()

    return SimpleNamespace(call=call, ran=ran, failing=failing, obj=obj, **paths)


def test_builds_once(build):
    assert build.call() == build.LIB
    assert sorted(build.ran) == ["ext.so", "lib.so", "unit.o"]
    build.call()
    assert build.ran == []


def test_library_without_torch(build, monkeypatch):
    """The C ABI needs no torch: a host without it gets the library."""
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.call() == build.LIB and build.LIB.exists()
    assert "ext.so" not in build.ran


def test_library_is_linked_when_the_extension_fails(build):
    build.failing.add("ext.so")
    with pytest.raises(RuntimeError, match="it failed"):
        build.call()
    assert build.LIB.exists()
    build.failing.clear()
    build.call()
    assert build.ran == ["ext.so"]


def test_library_is_linked_from_newer_objects(build):
    """Objects that a build compiled without linking them are linked by the next one."""
    build.call()
    later = build.LIB.stat().st_mtime + 10
    os.utime(build.obj, (later, later))
    build.call()
    assert build.ran == ["lib.so"]


def test_extension_follows_torch(build, monkeypatch):
    import torch

    build.call()
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".other")
    build.call()
    assert build.ran == ["ext.so"]
    build.call()
    assert build.ran == []
