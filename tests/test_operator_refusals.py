"""Refusals of the operators around the linear layer, on the CPU: argument
checks that need no device, in Python and at the C ABI."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kairo_b200 import _lib
from kairo_b200.ops import (
    BlockSparseLinear,
    QuantizedActivations,
    ScaledEmbedding,
    dequantize_activations,
    embedding_grad,
    embedding_lookup,
    quantize_activations,
    sort_tokens,
    sparse_linear_weight_grad,
)
from kairo_b200.types import BlockSparseMatrix


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


def _bsr():
    return BlockSparseMatrix(row_ptr=torch.tensor([0, 1], dtype=torch.int32), col_idx=torch.zeros(1, dtype=torch.int32),
                             blocks=torch.zeros(1, 64, 64), shape=(64, 64), block_size=(64, 64))


def test_checkpoint_refusals():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        quantize_activations(torch.zeros(4, 64))
    codes, steps = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(1, 4)
    q = QuantizedActivations(codes=codes, steps=steps, dtype=torch.float32)
    assert q.shape == (4, 64) and q.nbytes == 4 * 64 + 16
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        dequantize_activations(q)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        sparse_linear_weight_grad(torch.zeros(4, 64), q, _bsr())
    for bad in ({"codes": codes.to(torch.uint8)}, {"codes": codes[0]}, {"steps": steps.t()}, {"steps": steps.double()},
                {"codes": torch.zeros(4, 66, dtype=torch.int8)[:, 1:65]},     # rows not 16-byte aligned
                {"codes": torch.zeros(64, 4, dtype=torch.int8).t()}):
        with pytest.raises(ValueError):
            QuantizedActivations(**{"codes": codes, "steps": steps, "dtype": torch.float32, **bad})
    with pytest.raises(TypeError):
        QuantizedActivations(codes=codes, steps=steps, dtype=torch.float64)
    with pytest.raises(ValueError, match="checkpoint"):
        BlockSparseLinear(_bsr(), checkpoint="int4")


def test_checkpoint_c_refusals():
    lib = _lib.lib()
    some = ctypes.c_void_p(256)

    def quant(x=some, n=3, k=64, ldx=64, dt=0, codes=some, ldq=64, steps=some, lds=3):
        return lib.kairo_quantize_q8(x, n, k, ldx, dt, codes, ldq, steps, lds, None)

    def back(x=some, n=3, k=64, ldx=64, dt=0, codes=some, ldq=64, steps=some, lds=3):
        return lib.kairo_dequantize_q8(codes, ldq, steps, lds, n, k, x, ldx, dt, None)

    for fn in (quant, back):
        for kw in ({"x": None}, {"n": -1}, {"k": -1}, {"ldx": 63}, {"dt": 3}, {"codes": None}, {"ldq": 48},
                   {"ldq": 72}, {"steps": None}, {"lds": 2}, {"codes": ctypes.c_void_p(264)}):
            assert fn(**kw) == _lib.INVALID_VALUE, kw
        assert fn(n=0) == _lib.SUCCESS and fn(k=0) == _lib.SUCCESS
        assert fn(k=1 << 26, ldx=1 << 26, ldq=1 << 26) == _lib.NOT_SUPPORTED
    n = ctypes.c_size_t(0)
    d = _lib.KairoBsr(rows=64, cols=64, bm=64, bk=64, nbr=1, nnzb=1, nblocks_stored=1, dtype=_lib.DTYPE_BF16)
    d.col_idx = 256
    assert lib.kairo_bsr_sddmm_q8_workspace_size(None, 3, ctypes.byref(n)) == _lib.INVALID_VALUE
    assert lib.kairo_bsr_sddmm_q8_workspace_size(ctypes.byref(d), -1, ctypes.byref(n)) == _lib.INVALID_VALUE
    assert lib.kairo_bsr_sddmm_q8_workspace_size(ctypes.byref(d), 3, ctypes.byref(n)) == _lib.SUCCESS

    def wgrad(lddy=64, codes=some, ldq=64, steps=some, lds=3, out=some, odt=0, ws=some, wsb=n.value, dy=some):
        return lib.kairo_bsr_sddmm_q8(ctypes.byref(d), some, some, some, dy, lddy, codes, ldq, steps, lds, 3, out,
                                      odt, ws, wsb, None)

    for kw in ({"lddy": 63}, {"codes": None}, {"ldq": 40}, {"steps": None}, {"lds": 1}, {"out": None}, {"odt": 1},
               {"ws": None}, {"dy": None}):
        assert wgrad(**kw) == _lib.INVALID_VALUE, kw
    assert wgrad(wsb=n.value - 1) == _lib.WORKSPACE_TOO_SMALL
