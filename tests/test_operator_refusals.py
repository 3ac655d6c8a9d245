"""Refusals of the operators around the linear layer, on the CPU: argument
checks that need no device, in Python and at the C ABI."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kairo_b200 import _lib
from kairo_b200.ops import (
    AdapterPlan,
    AdaptedSparseLinear,
    BlockSparseLinear,
    LowRankAdapters,
    QuantizedActivations,
    ScaledEmbedding,
    adapter_linear,
    adapter_linear_backward,
    adapter_plan,
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
        return lib.kairo_embedding_grad_sorted(g, ldg, dt, some, some, nids, rows, dim, 1.0, out, ldo, odt, acc, ws,
                                               wsb, None)

    def grad_ids(ldg=8, dt=0, nids=3, rows=4, dim=8, ldo=8, odt=0, acc=1, ws=some, wsb=1 << 20, g=some, out=some,
                 ids=some, idb=8):
        return lib.kairo_embedding_grad(g, ldg, dt, ids, idb, nids, rows, dim, 1.0, out, ldo, odt, acc, ws, wsb, None)

    for fn in (grad, grad_ids):
        for kw in ({"ldg": 7}, {"ldo": 7}, {"dt": 3}, {"odt": 3}, {"nids": -1}, {"rows": -1}, {"dim": 0}, {"g": None},
                   {"nids": 1000, "ws": None}, {"out": None}):
            assert fn(**kw) == _lib.INVALID_VALUE, kw
        assert fn(nids=1000, wsb=10) == _lib.WORKSPACE_TOO_SMALL
    size = lib.kairo_embedding_grad_workspace_size
    assert size(-1, 8, 0, ctypes.byref(n)) == _lib.INVALID_VALUE and size(3, 8, 0, None) == _lib.INVALID_VALUE
    assert size(3, 8, 0, ctypes.byref(n)) == _lib.SUCCESS and n.value == 0  # a short list needs none
    assert size(3, 8, 1, ctypes.byref(n)) == _lib.SUCCESS and n.value > 0
    for fn in (grad, grad_ids):
        assert fn(nids=1 << 31) == _lib.NOT_SUPPORTED
        assert fn(rows=0) == _lib.SUCCESS
    assert grad_ids(ids=None) == _lib.INVALID_VALUE and grad_ids(idb=2) == _lib.INVALID_VALUE


def test_misaligned_memory_is_refused():
    """Workspaces and plans are bytes to the caller and vectors to the kernels."""
    lib = _lib.lib()
    some, odd, big = ctypes.c_void_p(256), ctypes.c_void_p(260), 1 << 30
    assert lib.kairo_token_sort(some, 8, 5000, 70000, some, some, odd, big, None) == _lib.INVALID_VALUE
    assert lib.kairo_embedding_grad(some, 8, 0, some, 8, 5000, 4, 8, 1.0, some, 8, 0, 0, odd, big,
                                    None) == _lib.INVALID_VALUE
    assert lib.kairo_embedding_grad_sorted(some, 8, 0, some, some, 300, 4, 8, 1.0, some, 8, 0, 0, odd, big,
                                           None) == _lib.INVALID_VALUE
    assert lib.kairo_adapter_plan_build(some, 8, 10, 3, odd, big, some, big, None) == _lib.INVALID_VALUE
    assert lib.kairo_adapter_plan_build(some, 8, 10, 3, some, big, odd, big, None) == _lib.INVALID_VALUE


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
        assert fn(k=1 << 28, ldx=1 << 28, ldq=1 << 28) == _lib.NOT_SUPPORTED
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


def test_adapter_refusals():
    down, up = torch.zeros(3, 8, 64, dtype=torch.bfloat16), torch.zeros(3, 8, 32, dtype=torch.bfloat16)
    a = LowRankAdapters(down=down, up=up)
    assert (a.count, a.rank, a.in_features, a.out_features) == (3, 8, 64, 32)
    for bad in ({"down": down[0]}, {"up": up[:2]}, {"up": up[:, :4]}, {"down": down.transpose(1, 2)},
                {"down": torch.zeros(3, 129, 64, dtype=torch.bfloat16), "up": torch.zeros(3, 129, 32,
                                                                                           dtype=torch.bfloat16)},
                {"down": down[:, :0], "up": up[:, :0]}, {"scale": torch.ones(2)},
                {"scale": torch.ones(3, dtype=torch.float64)}, {"scale": torch.ones(6)[::2]}):
        with pytest.raises(ValueError):
            LowRankAdapters(**{"down": down, "up": up, **bad})
    for bad in ({"down": down.half()}, {"down": down.float(), "up": up.float()}):
        with pytest.raises(TypeError):
            LowRankAdapters(**{"down": down, "up": up, **bad})
    plan = AdapterPlan(memory=torch.zeros(256, dtype=torch.uint8), num_tokens=4, num_adapters=3)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        adapter_plan(torch.zeros(4, dtype=torch.int64), 3)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        adapter_linear(torch.zeros(4, 64, dtype=torch.bfloat16), a, plan)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        adapter_linear_backward(torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(4, 64, dtype=torch.bfloat16), a,
                                plan)
    layer = BlockSparseLinear(_bsr())
    with pytest.raises(ValueError):
        AdaptedSparseLinear(layer, 0, 8)
    with pytest.raises(ValueError):
        AdaptedSparseLinear(layer, 2, 200)


def test_adapter_c_refusals():
    lib = _lib.lib()
    some = ctypes.c_void_p(256)
    a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    size = lib.kairo_adapter_plan_size
    assert size(10, 3, None, ctypes.byref(b)) == _lib.INVALID_VALUE
    assert size(-1, 3, ctypes.byref(a), ctypes.byref(b)) == _lib.INVALID_VALUE
    assert size(10, 65536, ctypes.byref(a), ctypes.byref(b)) == _lib.NOT_SUPPORTED
    assert size((1 << 24) + 1, 3, ctypes.byref(a), ctypes.byref(b)) == _lib.NOT_SUPPORTED
    assert size(10, 3, ctypes.byref(a), ctypes.byref(b)) == _lib.SUCCESS

    def build(ids=some, idb=8, plan=some, pb=a.value, ws=some, wb=b.value):
        return lib.kairo_adapter_plan_build(ids, idb, 10, 3, plan, pb, ws, wb, None)

    for kw in ({"ids": None}, {"idb": 1}, {"plan": None}, {"pb": a.value - 1}, {"ws": None}):
        assert build(**kw) == _lib.INVALID_VALUE, kw
    assert build(wb=b.value - 1) == _lib.WORKSPACE_TOO_SMALL

    def apply(x=some, ldx=64, k=64, down=some, up=some, n=32, rank=8, dt=2, plan=some, t=10, g=3, base=some, ldb=32,
              bdt=2, y=some, ldy=32, ydt=2, low=some):
        return lib.kairo_low_rank_apply(x, ldx, k, down, up, n, rank, dt, None, plan, t, g, base, ldb, bdt, y, ldy,
                                        ydt, low, None)

    for kw in ({"x": None}, {"ldx": 63}, {"k": 0}, {"down": None}, {"up": None}, {"n": 0}, {"rank": 0}, {"dt": 0},
               {"plan": None}, {"t": -1}, {"g": -1}, {"ldb": 31}, {"bdt": 1}, {"ldy": 31}, {"ydt": 1}, {"y": None, "low": None}):
        assert apply(**kw) == _lib.INVALID_VALUE, kw
    for kw in ({"rank": 129}, {"g": 65536}, {"t": (1 << 24) + 1}, {"k": (1 << 22) + 1, "ldx": 1 << 23}):
        assert apply(**kw) == _lib.NOT_SUPPORTED, kw
    assert apply(t=0) == _lib.SUCCESS

    def wgrad(low=some, rank=8, z=some, ldz=64, k=64, dt=2, plan=some, t=10, g=3, grad=some, gdt=0):
        return lib.kairo_low_rank_wgrad(low, rank, z, ldz, k, dt, plan, t, g, grad, gdt, None)

    for kw in ({"low": None}, {"rank": 0}, {"z": None}, {"ldz": 63}, {"k": 0}, {"dt": 0}, {"plan": None}, {"t": -1},
               {"g": -1}, {"grad": None}, {"gdt": 1}):
        assert wgrad(**kw) == _lib.INVALID_VALUE, kw
    def wgrad8(low=some, rank=8, q=some, ldq=64, steps=some, lds=10, k=64, dt=2, plan=some, t=10, g=3, grad=some, gdt=0):
        return lib.kairo_low_rank_wgrad_q8(low, rank, q, ldq, steps, lds, k, dt, plan, t, g, grad, gdt, None)

    for kw in ({"low": None}, {"rank": 0}, {"q": None}, {"ldq": 48}, {"ldq": 72}, {"steps": None}, {"lds": 9}, {"k": 0},
               {"dt": 0}, {"plan": None}, {"t": -1}, {"g": -1}, {"grad": None}, {"gdt": 1},
               {"q": ctypes.c_void_p(264)}):
        assert wgrad8(**kw) == _lib.INVALID_VALUE, kw
    def wgrads(dlow=some, low=some, rank=8, x=some, ldx=64, k=64, dy=some, lddy=32, n=32, dt=2, plan=some, t=10, g=3,
               dd=some, du=some, gdt=0):
        return lib.kairo_low_rank_wgrads(dlow, low, rank, x, ldx, k, dy, lddy, n, dt, plan, t, g, dd, du, gdt, None)

    for kw in ({"dlow": None}, {"low": None}, {"rank": 0}, {"x": None}, {"ldx": 63}, {"k": 0}, {"dy": None},
               {"lddy": 31}, {"n": 0}, {"dt": 0}, {"plan": None}, {"t": -1}, {"g": -1}, {"dd": None}, {"du": None},
               {"gdt": 1}):
        assert wgrads(**kw) == _lib.INVALID_VALUE, kw
    assert wgrads(rank=129) == _lib.NOT_SUPPORTED and wgrads(g=0) == _lib.SUCCESS
    assert wgrad(rank=129) == _lib.NOT_SUPPORTED and wgrad8(rank=129) == _lib.NOT_SUPPORTED
    assert wgrad(g=0) == _lib.SUCCESS
