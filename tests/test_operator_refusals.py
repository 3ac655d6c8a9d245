"""Refusals of the operators around the linear layer, on the CPU: argument
checks that need no device, in Python and at the C ABI."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kairo_b200 import _lib
from kairo_b200.ops import ScaledEmbedding, embedding_grad, embedding_lookup, sort_tokens


def test_embedding_needs_cuda_tensors():
    w, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        embedding_lookup(w, ids)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        embedding_grad(torch.zeros(3, 8), ids, 4)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        sort_tokens(ids, 4)
    with pytest.raises(ValueError):
        ScaledEmbedding(0, 8)


def test_embedding_c_refusals():
    """Every refusal comes before any device work, with a message."""
    lib = _lib.lib()
    n = ctypes.c_size_t(0)
    some = ctypes.c_void_p(256)  # never read: each call is refused first

    def lookup(rows=4, dim=8, ldw=8, dt=0, idb=8, nids=3, w=some, ids=some, out=some, odt=0):
        return lib.kairo_embedding_lookup(w, rows, dim, ldw, dt, ids, idb, nids, 1.0, out, odt, None)

    for kw in ({"rows": -1}, {"dim": 0}, {"ldw": 7}, {"dt": 9}, {"odt": -1}, {"idb": 2}, {"nids": -1}, {"w": None},
               {"ids": None}, {"out": None}):
        assert lookup(**kw) == _lib.INVALID_VALUE, kw
        assert lib.kairo_last_error_message()
    assert lookup(nids=0) == _lib.SUCCESS

    assert lib.kairo_token_sort_workspace_size(-1, 5, ctypes.byref(n)) == _lib.INVALID_VALUE
    assert lib.kairo_token_sort_workspace_size(1 << 31, 5, ctypes.byref(n)) == _lib.NOT_SUPPORTED
    assert lib.kairo_token_sort_workspace_size(5, 1 << 31, ctypes.byref(n)) == _lib.NOT_SUPPORTED
    assert lib.kairo_token_sort_workspace_size(5000, 70000, ctypes.byref(n)) == _lib.SUCCESS
    assert lib.kairo_token_sort(some, 8, 5000, 70000, some, some, some, n.value - 1, None) == _lib.WORKSPACE_TOO_SMALL
    assert lib.kairo_token_sort(some, 3, 5000, 70000, some, some, some, n.value, None) == _lib.INVALID_VALUE
    assert lib.kairo_token_sort(None, 8, 5000, 70000, some, some, some, n.value, None) == _lib.INVALID_VALUE
    assert lib.kairo_token_sort(None, 8, 0, 70000, None, None, None, n.value, None) == _lib.SUCCESS

    def grad(ldg=8, dt=0, nids=3, rows=4, dim=8, ldo=8, odt=0, acc=1, ws=some, wsb=1 << 20, g=some, out=some):
        return lib.kairo_embedding_grad(g, ldg, dt, some, some, nids, rows, dim, 1.0, out, ldo, odt, acc, ws, wsb,
                                        None)

    for kw in ({"ldg": 7}, {"ldo": 7}, {"dt": 3}, {"odt": 3}, {"nids": -1}, {"rows": -1}, {"dim": 0}, {"g": None},
               {"ws": None}, {"out": None}):
        assert grad(**kw) == _lib.INVALID_VALUE, kw
    assert grad(wsb=10) == _lib.WORKSPACE_TOO_SMALL
    assert grad(nids=1 << 31) == _lib.NOT_SUPPORTED
    assert grad(rows=0) == _lib.SUCCESS
