"""The compiled module beside the library is optional: where it cannot be built the library is, and it is built anew for another torch."""
import os
import types

import pytest
import torch

from flaggems_sglang_b200 import build as b


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A package of one kernel file and one module source, with a C++ compiler that notes its calls, or fails where `broken` is there."""
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (csrc / "a.cu").write_text('extern "C" int one() { return 1; }\n')
    (csrc / "host.cpp").write_text("\n")
    cxx = tmp_path / "cxx"
    cxx.write_text(f'#!/bin/sh\n[ -e {tmp_path}/broken ] && {{ echo cannot; exit 1; }}\necho "$@" >> {tmp_path}/calls\n'
                   'while [ "$1" != -o ]; do shift; done; echo module > "$2"\n')
    cxx.chmod(0o755)
    monkeypatch.setenv("CXX", str(cxx))
    for name, path in dict(CSRC=csrc, OBJ_DIR=tmp_path / "obj", LIB_PATH=tmp_path / "lib.so", HOST_SRC=csrc / "host.cpp",
                           HOST_PATH=tmp_path / "_host.so").items():
        monkeypatch.setattr(b, name, str(path))
    return tmp_path


def calls(tree):
    path = tree / "calls"
    return len(path.read_text().splitlines()) if path.exists() else 0


def test_library_is_built_where_the_module_is_not(tree, capfd):
    (tree / "broken").write_text("")
    (tree / "_host.so").write_text("of another build")
    os.utime(tree / "_host.so", (1, 1))
    assert b.build() == str(tree / "lib.so") and (tree / "lib.so").exists()
    assert not (tree / "_host.so").exists()
    assert "cannot" in capfd.readouterr().err
    os.remove(tree / "broken")
    b.build()
    assert (tree / "_host.so").exists()


def test_library_is_built_without_torch(tree, monkeypatch):
    monkeypatch.setitem(__import__("sys").modules, "torch", None)
    assert os.path.exists(b.build())
    assert calls(tree) == 0


def test_module_is_built_anew_for_another_torch(tree, monkeypatch):
    b.build()
    b.build()
    assert calls(tree) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.0")
    b.build()
    b.build()
    assert calls(tree) == 2


def test_module_of_another_torch_is_not_used_and_says_so(monkeypatch):
    import flaggems_sglang_b200 as fg
    from flaggems_sglang_b200 import _C

    _C.lib()
    monkeypatch.setattr(fg, "_host", types.SimpleNamespace(torch_version="0.0.0"), raising=False)
    monkeypatch.setattr(_C, "_host", None)
    with pytest.warns(RuntimeWarning, match="0.0.0"):
        assert _C.host() is False
