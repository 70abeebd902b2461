"""The library is built and linked whatever becomes of the Python entries (which need torch's and Python's headers)."""

import importlib.util

import pytest

from myinfer_b200 import build as b

needs_nvcc = pytest.mark.skipif(not any(c and b.Path(c).exists() for c in (b.os.environ.get("NVCC"), b.shutil.which("nvcc"),
                                                                     "/usr/local/cuda/bin/nvcc")), reason="no nvcc")


@pytest.fixture
def tree(tmp_path, monkeypatch):
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "one.cu").write_text('extern "C" __attribute__((visibility("default"))) int one() { return 1; }')
    for name, path in (("CSRC", "csrc"), ("OBJ", "obj"), ("LIB", "libone.so"), ("BINDING", "_binding.so")):
        monkeypatch.setattr(b, name, tmp_path / path)
    return tmp_path


@needs_nvcc
def test_library_without_the_binding(tree, monkeypatch):
    def fail():
        raise RuntimeError("tree_binding.cpp: Python.h: no such file")
    monkeypatch.setattr(b, "build_binding", fail)
    with pytest.raises(RuntimeError, match="Python.h"):  # the package's tree operators do need it
        b.build()
    assert (tree / "libone.so").exists()


@needs_nvcc
def test_library_without_torch(tree, monkeypatch):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert b.build() == tree / "libone.so" and b.LIB.exists() and not b.BINDING.exists()
