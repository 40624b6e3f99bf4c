"""What is built, in which order, and for whom (CPU, no compiler is run)."""
import importlib.util
import os
import sysconfig

import pytest
import torch

from kvcomp_b200 import build


@pytest.fixture
def runs(monkeypatch, tmp_path):
    """The files that compilers would write, in order; they are written."""
    made = []

    def run(cmd, to, verbose):
        made.append(os.path.basename(to).split(".")[0])
        open(to, "w").close()
        return to
    monkeypatch.setattr(build, "_run", run)
    monkeypatch.setattr(build, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "libkvcomp_b200.so"))
    return made


def test_the_library_comes_first_and_needs_no_torch(runs, monkeypatch):
    assert build.build(binding=False) == build.LIB and runs == ["libkvcomp_b200"]
    build.build()
    assert runs == ["libkvcomp_b200", "kvc_torch"]
    build.build()
    assert len(runs) == 2
    build.build(force=True)
    assert runs[2:] == ["libkvcomp_b200", "kvc_torch"]


def test_without_torch(runs, monkeypatch, capsys):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert build.build() == build.LIB and runs == ["libkvcomp_b200"]
    assert "kvc_torch" in capsys.readouterr().err


def test_a_binding_that_cannot_be_built_leaves_the_library(runs, monkeypatch):
    monkeypatch.setattr(build, "build_binding", lambda *a: (_ for _ in ()).throw(RuntimeError("no headers")))
    with pytest.raises(RuntimeError):
        build.build()
    assert runs == ["libkvcomp_b200"]


@pytest.mark.parametrize("other", [lambda m: m.setattr(torch, "__version__", "9.9.9+cu999"), lambda m: m.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI),
                                   lambda m: m.setattr(sysconfig, "get_config_var", lambda name: "cpython-999")], ids=["torch", "abi", "python"])
def test_a_binding_of_another_torch_or_python_is_not_taken(runs, monkeypatch, other):
    path = build.build_binding()
    assert not build.binding_is_stale() and build.build_binding() == path and len(runs) == 1
    other(monkeypatch)
    assert build.binding_is_stale() and build.build_binding() != path and len(runs) == 2
    monkeypatch.undo()
