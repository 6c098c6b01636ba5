"""What build() needs and when it builds again, with compilers that only write their output files."""
import importlib.metadata
import os
import sys

import pytest

FAKE = "#!/bin/sh\nwhile [ $# -gt 0 ]; do if [ \"$1\" = -o ]; then echo built > \"$2\"; fi; shift; done\necho \"$0\" >> {log}\n"


@pytest.fixture
def tree(lib, tmp_path, monkeypatch):
    """The package pointed at a source folder of its own."""
    csrc, log = tmp_path / "csrc", tmp_path / "log"
    csrc.mkdir()
    log.write_text("")
    for name in ("a.cu", "tensors.cpp"):
        (csrc / name).write_text("")
    for name, value in dict(CSRC=str(csrc), LIB_PATH=str(tmp_path / "lib.so"), TENSORS_PATH=str(tmp_path / "_tensors.so"), SOURCES=["a.cu"]).items():
        monkeypatch.setattr(lib, name, value)
    for variable in ("NVCC", "CXX"):
        compiler = tmp_path / variable.lower()
        compiler.write_text(FAKE.format(log=log))
        compiler.chmod(0o755)
        monkeypatch.setenv(variable, str(compiler))

    def runs():
        """The compilers that ran since the last look."""
        lines = [os.path.basename(line) for line in log.read_text().split()]
        log.write_text("")
        return lines
    tree.runs = runs
    return tree


def test_the_c_library_needs_nvcc_alone(lib, tree, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)                 # what an import finds where there is no torch
    assert lib.build() == lib.LIB_PATH and os.path.exists(lib.LIB_PATH) and not os.path.exists(lib.TENSORS_PATH)
    assert tree.runs() == ["nvcc", "nvcc"]                          # one source, one link


def test_a_missing_c_compiler_leaves_the_c_library(lib, tree, monkeypatch):
    monkeypatch.setenv("CXX", str(lib.CSRC) + "/no-such-compiler")
    with pytest.raises(lib.B200RLError, match="C\\+\\+ compiler"):
        lib.build()
    assert os.path.exists(lib.LIB_PATH) and not os.path.exists(lib.TENSORS_PATH)


def test_another_torch_or_python_builds_the_tensor_calls_again(lib, tree, monkeypatch):
    lib.build()
    assert tree.runs() == ["nvcc", "nvcc", "cxx"]
    lib.build()
    assert tree.runs() == []
    version = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0.1" if name == "torch" else version(name))
    lib.build()
    assert tree.runs() == ["cxx"]
    lib.build()
    assert tree.runs() == []
    monkeypatch.setattr(sys, "version", "another Python")
    lib.build()
    assert tree.runs() == ["cxx"]
