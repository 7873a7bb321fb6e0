"""The build's two artefacts on their own: the library, and the host part that may be missing.  Nothing is compiled here."""
import importlib.util
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(tmp_path, monkeypatch):
    """moa_b200/build.py with its artefacts in a folder of their own, and a subprocess.run that writes what it is asked for."""
    spec = importlib.util.spec_from_file_location("_build_under_test", os.path.join(ROOT, "moa_b200", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    real, module.ran, module.broken = module.HOST, [], None
    monkeypatch.setattr(module, "LIB", str(tmp_path / "libmoa_b200.so"))
    monkeypatch.setattr(module, "HOST", str(tmp_path / os.path.basename(real)))
    monkeypatch.setattr(module, "_nvcc", lambda: "/cuda/bin/nvcc")

    def run(cmd, check):
        kind = "nvcc" if cmd[0].endswith("nvcc") else "host"
        module.ran.append(kind)
        if kind == "host" and module.broken is not None:
            raise module.broken
        out = cmd[cmd.index("-o") + 1]
        if not out.endswith(".o"):
            open(out, "w").close()

    monkeypatch.setattr(module.subprocess, "run", run)
    return module


def test_each_artefact_is_made_when_it_is_stale(build):
    assert build.build() == build.LIB
    assert set(build.ran) == {"nvcc", "host"} and os.path.exists(build.LIB) and os.path.exists(build.HOST)
    build.ran.clear()
    build.build()
    assert build.ran == []
    os.remove(build.HOST)
    build.build()                                         # the host part alone: no kernel is compiled for it
    assert build.ran == ["host"]
    build.ran.clear()
    os.remove(build.LIB)
    build.build()
    assert "host" not in build.ran and "nvcc" in build.ran
    build.ran.clear()
    build.build(force=True)
    assert set(build.ran) == {"nvcc", "host"}


@pytest.mark.parametrize("broken", [subprocess.CalledProcessError(1, "g++"), FileNotFoundError("g++")])
def test_the_library_is_built_where_the_host_part_cannot_be(build, broken):
    build.build()
    os.utime(build.HOST, (1, 1))                          # of an older source
    build.broken = broken
    with pytest.warns(RuntimeWarning, match="host part"):
        assert build.build(force=True) == build.LIB
    assert not os.path.exists(build.HOST)                 # the older one is not left to be loaded
    build.ran.clear()
    with pytest.warns(RuntimeWarning, match="host part"):
        build.build()
    assert build.ran == ["host"]


def test_the_host_part_is_for_this_python_and_this_torch(build):
    from moa_b200 import paged

    name = os.path.basename(build.HOST)
    assert name == os.path.basename(paged.HOST_PATH) and paged.HOST_PATH.startswith(os.path.join(ROOT, "moa_b200"))
    assert sys.implementation.cache_tag in name and torch.__version__ in name
    assert paged._host is not None and paged._host.__file__ == paged.HOST_PATH


def test_a_host_part_of_another_library_is_not_used(monkeypatch):
    from moa_b200 import _lib, paged

    assert paged._load_host() is not None
    monkeypatch.setattr(_lib, "ABI_VERSION", _lib.ABI_VERSION + 1)
    assert paged._load_host() is None
    monkeypatch.undo()
    monkeypatch.setattr(paged, "HOST_PATH", paged.HOST_PATH + ".not")
    assert paged._load_host() is None
