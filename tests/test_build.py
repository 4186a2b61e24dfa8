"""The build of the Python extension beside the C library (build.py)."""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(tmp_path, monkeypatch):
    """build.py with the extension's path moved and its commands recorded in
    `ran` (each makes its output file)."""
    spec = importlib.util.spec_from_file_location("fb2_build_under_test", os.path.join(ROOT, "forge-lm_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.ran = []

    def run(cmd, **_):
        mod.ran.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass

    monkeypatch.setattr(mod, "BINDING", str(tmp_path / "_serving.so"))
    monkeypatch.setattr(mod.subprocess, "run", run)
    return mod


def test_the_library_builds_without_torch(build, monkeypatch):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    # the library is up to date (nothing here may write it)
    monkeypatch.setattr(build, "gen_fixups", lambda *a: None)
    monkeypatch.setattr(build, "read_stamp", lambda: {"flags": build._flags()})
    monkeypatch.setattr(build, "_newer", lambda target, sources: target == build.BINDING)
    assert build.build_binding() is None
    assert build.build() == build.LIB
    assert build.ran == [] and not os.path.exists(build.BINDING)


def test_the_extension_is_built_again_for_another_torch(build, monkeypatch):
    pytest.importorskip("torch")
    assert build.build_binding() == build.BINDING and len(build.ran) == 1
    assert build.build_binding() == build.BINDING and len(build.ran) == 1  # up to date
    real = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0.1" if name == "torch" else real(name))
    build.build_binding()
    assert len(build.ran) == 2
    build.build_binding()
    assert len(build.ran) == 2
    os.remove(build.stamp_path(build.BINDING))  # one whose torch is not known
    build.build_binding()
    assert len(build.ran) == 3


def test_an_extension_for_another_torch_is_not_loaded(pkg, monkeypatch):
    pytest.importorskip("torch")
    from forge_lm_b200 import serving
    monkeypatch.setattr(serving, "_calls", None)
    assert serving._load() is not None
    monkeypatch.setattr(serving, "_calls", None)
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0.1")
    with pytest.raises(OSError, match="another|installed"):
        serving._load()


def test_an_extension_without_its_record_is_loaded(pkg, monkeypatch, tmp_path):
    pytest.importorskip("torch")
    from forge_lm_b200 import serving
    lone = tmp_path / "_serving.so"
    lone.symlink_to(serving._PATH)
    monkeypatch.setattr(serving, "_PATH", str(lone))
    monkeypatch.setattr(serving, "_calls", None)
    assert serving._load() is not None
