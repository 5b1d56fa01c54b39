"""CPU tests of the kernels' build (ops/build.py): what is built where."""

import importlib.util

import pytest

from code_interpreter_amd.ops import build


@pytest.fixture
def compiled(monkeypatch):
    done = []
    monkeypatch.setattr(build, "_compile",
                        lambda out, sources, verbose: done.append(out))
    return done


def test_without_torch_the_other_modules_are_built(compiled, monkeypatch,
                                                   capsys):
    find = importlib.util.find_spec
    monkeypatch.setattr(
        importlib.util, "find_spec",
        lambda name, *a: None if name == "torch" else find(name, *a))
    assert build.build(force=True) == build.OUTPUT
    assert compiled == [build.OUTPUT, build.GEMM_OUTPUT]
    assert "_hiplm.so is not built" in capsys.readouterr().out


def test_next_to_a_torch_without_rocm(compiled, monkeypatch, tmp_path):
    (tmp_path / "torch" / "lib").mkdir(parents=True)
    (tmp_path / "torch" / "__init__.py").touch()
    spec = importlib.util.spec_from_file_location(
        "torch", tmp_path / "torch" / "__init__.py",
        submodule_search_locations=[str(tmp_path / "torch")])
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: spec)
    build.build(force=True)
    assert compiled == [build.OUTPUT, build.GEMM_OUTPUT]
    (tmp_path / "torch" / "lib" / "libtorch_hip.so").touch()
    build.build(force=True)
    assert compiled[2:] == [out for out, _ in build.MODULES]


def test_a_module_that_cannot_be_built_is_not_out_of_date(monkeypatch):
    monkeypatch.setattr(build, "_torch_dir", lambda: None)
    monkeypatch.setattr(build, "_needs",
                        lambda out, sources: out == build.LM_OUTPUT)
    assert not build.needs_build()
