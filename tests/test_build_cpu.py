"""The build without a compiler run: the C library needs nvcc alone, its Python binding more."""

from __future__ import annotations

import pytest

from kta_b200 import build


@pytest.fixture
def made(monkeypatch, tmp_path):
    """build() with the library as it is, and a binding of an earlier build in a folder of the test."""
    monkeypatch.setattr(build, "_build_library", lambda verbose, ptxas: build.LIB, raising=False)
    monkeypatch.setattr(build, "BINDING", tmp_path / "_binding.so")
    monkeypatch.setattr(build, "BUILD", tmp_path)
    for name in ("_binding.so", "binding.hash"):
        (tmp_path / name).write_text("of an earlier build")
    calls = []
    monkeypatch.setattr(build, "_run", lambda cmd, what, verbose: calls.append(cmd))
    return calls


@pytest.mark.parametrize("what", ["torch", "torch's CUDA libraries", "g++", "Python.h"])
def test_without_the_bindings_needs_the_library_is_built(made, monkeypatch, tmp_path, capsys, what):
    real = build.importlib.util.find_spec
    if what == "torch":
        monkeypatch.setattr(build.importlib.util, "find_spec", lambda n: None if n == "torch" else real(n))
    elif what == "torch's CUDA libraries":
        spec = type("Spec", (), {"submodule_search_locations": [str(tmp_path)]})
        monkeypatch.setattr(build.importlib.util, "find_spec", lambda n: spec if n == "torch" else real(n))
    elif what == "g++":
        which = build.shutil.which
        monkeypatch.setattr(build.shutil, "which", lambda n: None if n == "g++" else which(n))
    else:
        paths = {**build.sysconfig.get_paths(), "include": str(tmp_path)}
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: paths)
    assert build.build() == build.LIB
    assert made == []
    assert not build.BINDING.exists()  # an earlier one may be of another ABI: loading it has to fail
    said = capsys.readouterr().err
    assert "binding not built" in said and what in said


def test_a_compiler_error_of_the_binding_is_an_error(made, monkeypatch):
    def fails(cmd, what, verbose):
        raise RuntimeError(f"{what} failed")

    assert build.build() == build.LIB and len(made) == 1 and "binding.cpp" in " ".join(made[0])
    (build.BUILD / "binding.hash").unlink()
    monkeypatch.setattr(build, "_run", fails)
    with pytest.raises(RuntimeError, match="binding"):
        build.build()
