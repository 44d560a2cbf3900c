"""The build of the module that describes torch tensors: where it cannot be built the rest of the build goes on and the
Python form is used; a module of another Python, torch or source is not. CPU only."""
import os
import shutil
import sysconfig

import pytest

from kore_b200 import build
from kore_b200 import paged as P

torch = pytest.importorskip("torch")


@pytest.fixture
def elsewhere(tmp_path, monkeypatch):
    """The package's folder, with the sources and a module as the build leaves it."""
    built = build.build_tensors()
    monkeypatch.setattr(build, "PKG", str(tmp_path))
    monkeypatch.setattr(build, "TENSORS", str(tmp_path / os.path.basename(build.TENSORS)))
    if built:
        shutil.copy(built, build.TENSORS)
    return tmp_path


@pytest.mark.parametrize("cxx", ["/nowhere/g++", "false"])
def test_without_a_compiler_there_is_no_module_and_no_failure(elsewhere, monkeypatch, capfd, cxx):
    monkeypatch.setenv("CXX", cxx)
    assert build.build_tensors(force=True) is None
    assert os.listdir(elsewhere) == []   # an earlier one would not be of these sources
    assert "described in Python" in capfd.readouterr().err


def test_without_pythons_headers(elsewhere, monkeypatch, capfd):
    paths = sysconfig.get_paths()
    monkeypatch.setattr(sysconfig, "get_paths", lambda: {**paths, "include": str(elsewhere / "none")})
    assert build.build_tensors(force=True) is None
    assert os.listdir(elsewhere) == []


def test_the_module_is_named_for_its_python():
    """Another Python does not import it: it has another suffix."""
    assert os.path.basename(build.TENSORS) == "_tensors" + sysconfig.get_config_var("EXT_SUFFIX") != "_tensors.so"


def test_an_untagged_module_is_taken_away(elsewhere, monkeypatch):
    (elsewhere / "_tensors.so").write_bytes(b"")
    monkeypatch.setenv("CXX", "false")   # (nothing is compiled: the module is as the sources want it)
    assert build.build_tensors() == build.TENSORS
    assert os.listdir(elsewhere) == [os.path.basename(build.TENSORS)]


def test_a_module_of_another_torch_is_stale(elsewhere):
    version = torch.__version__.split("+")[0]
    assert not build._tensors_stale([], version)
    assert build._tensors_stale([], "1." + version)
    assert build._tensors_stale([], version + ".1")
    os.remove(build.TENSORS)
    assert build._tensors_stale([], version)


def test_a_module_of_another_torch_is_not_used(monkeypatch):
    monkeypatch.setattr(P, "_rows_in", P._rows_of)
    monkeypatch.setattr(P, "_ints_in", P._ints_of)
    monkeypatch.setattr(torch, "__version__", "0.1")
    P._import_torch()
    assert not P._describe_natively() and P._rows_in is P._rows_of and P._ints_in is P._ints_of
