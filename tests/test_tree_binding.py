"""The compiled Python entries of the tree operators: errors, without a device."""

import ctypes

import pytest
import torch

from myinfer_b200 import _lib, tree


def test_errors():
    b = tree._load()
    cpu = torch.zeros(2, 3, dtype=torch.int32)
    for call, text in ((lambda: tree.tree_plan(cpu), "int32 CUDA tensor"), (lambda: tree.tree_accept(None, cpu, cpu), "must be a tensor"),
                       (lambda: tree.process_logits(cpu.float()), "bf16 or fp32 CUDA"),
                       (lambda: tree.tree_attention(cpu, cpu, cpu, cpu, cpu, 1.0), "bf16 CUDA"),
                       # numbers in the text: the binding and torch must share one C++ library
                       (lambda: b.commit(16, 1, 2, 1, 128, 0, cpu, torch.zeros(2, 65, dtype=torch.int32), cpu), "path must be int32 .2, 1 to 64"),
                       (lambda: b.commit(16, 1, 2, 1, 128, 0, cpu, cpu, cpu), "lengths must be .* of shape .2. on cuda:0")):
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(TypeError, match="expected 4 arguments, got 1"):
        b.accept(cpu)
    with pytest.raises(ValueError, match="invalid literal"):
        b.commit(16, "x", 2, 1, 128, 0, cpu, cpu, cpu)
    with pytest.raises(ValueError, match="null entry point"):
        b.bind(0, 0, 0, 0, 0, 0, None)


def test_bound_entries():
    L = _lib.lib()
    assert all(ctypes.cast(getattr(L, n), ctypes.c_void_p).value for n in tree._ENTRIES)
    assert set(tree._ENTRIES) <= set(_lib.header_symbols())
