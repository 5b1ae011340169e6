"""The build without torch, with another torch, and with a source that does not compile."""
import importlib
import os
import subprocess
import sys

import pytest


@pytest.fixture()
def build(pkg, monkeypatch, tmp_path):
    b = importlib.import_module("faster_rwkv_b200.build")
    monkeypatch.setattr(b, "TORCH_LIB", str(tmp_path / "ext.so"))
    monkeypatch.setattr(b, "TORCH_STAMP", str(tmp_path / "stamp.txt"), raising=False)
    monkeypatch.setattr(b, "SOURCES", [])
    return b


def test_the_library_is_built_without_torch(build, monkeypatch):
    """what the torch entry alone needs stops nothing else"""
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build_lib() == build.LIB
    assert not os.path.exists(build.TORCH_LIB)


def test_another_torch_rebuilds_the_entry(build, monkeypatch):
    built = []

    class Gxx:
        pid, returncode = -1, 0

        def __init__(self, cmd, **kw):
            built.append(cmd)
            out = cmd[cmd.index("-o") + 1]
            with open(out, "w") as f:
                f.write("ext")

        def communicate(self):
            return "", None

    monkeypatch.setattr(subprocess, "Popen", Gxx)
    build.build_lib()
    assert len(built) == 1 and os.path.exists(build.TORCH_LIB)
    build.build_lib()
    assert len(built) == 1
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0.1")
    build.build_lib()
    assert len(built) == 2
    build.build_lib()
    assert len(built) == 2


def test_a_source_that_does_not_compile_leaves_no_compiler_running(build, monkeypatch, tmp_path):
    """nvcc fails (a stand-in that exits with 1): the compiler of the torch entry is ended and waited for, and no half of its output is taken"""
    g = subprocess.Popen([sys.executable, "-c", "import time; time.sleep(60)"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, start_new_session=True)
    monkeypatch.setattr(build, "_start_torch", lambda force: g)
    (tmp_path / "nvcc").write_text("#!/bin/sh\nexit 1\n")
    (tmp_path / "nvcc").chmod(0o755)
    monkeypatch.setenv("PATH", str(tmp_path) + os.pathsep + os.environ["PATH"])
    monkeypatch.setattr(build, "SOURCES", ["broken.cu"])
    monkeypatch.setattr(build, "CSRC", str(tmp_path))
    (tmp_path / "broken.cu").write_text("no C++\n")
    with pytest.raises(RuntimeError, match="broken.cu"):
        build.build_lib()
    assert g.poll() is not None
    assert not os.path.exists(build.TORCH_LIB)
