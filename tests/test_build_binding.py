"""The tensor binding is the only part of the build that needs torch: a torch
that it cannot be built against leaves the rest of the build as it is."""
import importlib.machinery
import os
import shutil

import pytest

import build as pkg_build


@pytest.fixture
def lib(tmp_path, monkeypatch):
    """The built libraries in a folder of their own, all but the binding up to date."""
    pkg_build.build()
    at = tmp_path / "lib"
    shutil.copytree(pkg_build.LIB, at)
    monkeypatch.setattr(pkg_build, "LIB", str(at))
    monkeypatch.setattr(pkg_build, "OBJ", str(at / "obj"))
    return at


def fake_torch(monkeypatch, root):
    """A torch that is found, but has neither CUDA headers nor libraries."""
    (root / "include").mkdir(parents=True)
    (root / "lib").mkdir()
    (root / "version.py").write_text("__version__ = '0'\n")
    os.utime(root / "version.py", (2**31, 2**31))  # newer than any binding
    spec = importlib.machinery.ModuleSpec("torch", None, is_package=True)
    spec.submodule_search_locations = [str(root)]
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda n, *a: spec if n == "torch" else find(n, *a))


def test_a_torch_without_cuda_leaves_the_rest_of_the_build(lib, tmp_path, monkeypatch, capfd):
    fake_torch(monkeypatch, tmp_path / "torch")
    out = pkg_build.build()
    assert "dev" not in out and not (lib / "_myos_dev.so").exists()  # nor one of another torch
    assert all(os.path.exists(out[k]) for k in ("cuda", "synth", "cli"))
    assert "myos.dev is left out" in capfd.readouterr().err


def test_without_torch_the_binding_is_left_out(lib, monkeypatch):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda n, *a: None if n == "torch" else find(n, *a))
    out = pkg_build.build()
    assert "dev" not in out and os.path.exists(out["cuda"])


def test_a_failing_step_of_the_rest_still_raises(lib, monkeypatch):
    def no(cmd):
        raise RuntimeError("build step failed")

    monkeypatch.setattr(pkg_build, "_run", no)
    os.remove(lib / "libmyos_synth.so")
    with pytest.raises(RuntimeError):
        pkg_build.build()
