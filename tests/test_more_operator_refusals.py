"""Refusals of the vocabulary loss and the gated projection, on the CPU: argument checks that need no
device, in Python and at the C ABI."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kairo_b200 import _lib
from kairo_b200.ops import (
    GatedWeights,
    LinearCrossEntropy,
    ScaledEmbedding,
    gated_weights,
    linear_cross_entropy,
    linear_cross_entropy_backward,
    sparse_gated_linear,
    sparse_gated_linear_backward,
)
from kairo_b200.ops import gated as gated_module
from kairo_b200.ops import vocab_loss as loss_module
from kairo_b200.types import BlockSparseMatrix

BF16 = torch.bfloat16


def test_loss_needs_cuda_tensors():
    x, w, ids = torch.zeros(3, 8, dtype=BF16), torch.zeros(5, 8, dtype=BF16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        linear_cross_entropy(x, w, ids)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        linear_cross_entropy_backward(torch.ones(()), x, w, ids, torch.zeros(3))


def test_loss_arguments():
    x, w, ids = torch.zeros(3, 8, dtype=BF16), torch.zeros(5, 8, dtype=BF16), torch.zeros(3, dtype=torch.int64)

    def problem(x=x, w=w, ids=ids, reduction="mean"):
        return loss_module._problem("op", x, w, ids, reduction)

    assert problem()[3:] == (3, 5, 8, _lib.DTYPE_BF16, 2)
    for kw in ({"reduction": "avg"}, {"w": w[0]}, {"w": w[:0]}, {"x": x[:2]}, {"x": x[:, :7]}, {"ids": ids[:2]},
               {"ids": ids.view(3, 1)}):
        with pytest.raises(ValueError):
            problem(**kw)
    for kw in ({"x": x.half()}, {"x": x.float(), "w": w.float()}, {"ids": ids.float()}, {"ids": ids.short()}):
        with pytest.raises(TypeError):
            problem(**kw)
    with pytest.raises(ValueError, match="dw must be"):
        loss_module._gradient("op", "dw", torch.zeros(5, 9, dtype=BF16), w, 5, 8)
    with pytest.raises(ValueError, match="dw must be"):
        loss_module._gradient("op", "dw", torch.zeros(8, 5, dtype=BF16).t(), w, 5, 8)
    with pytest.raises(ValueError, match="must not share memory"):
        loss_module._gradient("op", "dw", w, w, 5, 8, w)


def test_loss_module_arguments():
    with pytest.raises(TypeError):
        LinearCrossEntropy(torch.zeros(4, 8, dtype=BF16))
    with pytest.raises(TypeError):
        LinearCrossEntropy(torch.nn.Parameter(torch.zeros(4, 8)))
    with pytest.raises(ValueError):
        LinearCrossEntropy(torch.nn.Parameter(torch.zeros(4, 8, dtype=BF16)), reduction="max")
    emb = ScaledEmbedding(4, 8, dtype=BF16)
    assert LinearCrossEntropy(emb).weight is emb.weight


def test_loss_c_refusals():
    """Every refusal comes before any device work, with a message."""
    lib = _lib.lib()
    some = ctypes.c_void_p(256)  # never read: each call is refused first
    n = ctypes.c_size_t(0)

    def size(tokens=3, vocab=5, dim=8, ldx=8, ldw=8):
        return lib.kairo_vocab_loss_workspace_size(some, ldx, some, ldw, tokens, vocab, dim, ctypes.byref(n))

    assert size() == _lib.SUCCESS and n.value >= 256
    small = n.value
    assert size(vocab=50_000) == _lib.SUCCESS and n.value > small
    for kw in ({"tokens": -1}, {"vocab": 0}, {"dim": 0}, {"ldx": 7}, {"ldw": 7}):
        assert size(**kw) == _lib.INVALID_VALUE, kw
        assert lib.kairo_last_error_message()
    assert size(tokens=1 << 31) == _lib.NOT_SUPPORTED
    assert size(tokens=1 << 30, vocab=1 << 30) == _lib.NOT_SUPPORTED
    assert lib.kairo_vocab_loss_workspace_size(some, 8, some, 8, 3, 5, 8, None) == _lib.INVALID_VALUE

    def loss(x=some, w=some, ids=some, idb=8, dt=_lib.DTYPE_BF16, red=2, out=some, lse=some, ws=some, nbytes=1 << 30,
             err=some, tokens=3, ldx=8):
        return lib.kairo_vocab_loss(x, ldx, w, 8, tokens, 5, 8, dt, ids, idb, 1.0, red, out, lse, ws, nbytes, err, None)

    for kw in ({"x": None}, {"w": None}, {"ids": None}, {"out": None}, {"lse": None}, {"ws": None}, {"err": None},
               {"idb": 2}, {"dt": _lib.DTYPE_F32}, {"dt": 7}, {"red": 3}, {"red": -1}, {"ws": ctypes.c_void_p(264)},
               {"ldx": 7}):
        assert loss(**kw) == _lib.INVALID_VALUE, kw
    assert loss(nbytes=300) == _lib.WORKSPACE_TOO_SMALL
    assert loss(tokens=0, red=0) == _lib.SUCCESS

    def back(grad=some, x=some, w=some, ids=some, lse=some, dx=some, dw=some, ws=some, nbytes=1 << 30, err=some,
             lddx=8, lddw=8, tokens=3, red=2):
        return lib.kairo_vocab_loss_backward(grad, x, 8, w, 8, tokens, 5, 8, _lib.DTYPE_F16, ids, 8, 1.0, red, lse, dx,
                                             lddx, dw, lddw, ws, nbytes, err, None)

    for kw in ({"grad": None}, {"x": None}, {"w": None}, {"ids": None}, {"lse": None}, {"ws": None}, {"err": None},
               {"lddx": 7}, {"lddw": 7}, {"red": 9}, {"ws": ctypes.c_void_p(264)}):
        assert back(**kw) == _lib.INVALID_VALUE, kw
    assert back(nbytes=300) == _lib.WORKSPACE_TOO_SMALL
    assert back(dx=None, dw=None) == _lib.SUCCESS  # nothing to compute
    assert back(tokens=0, dw=None) == _lib.SUCCESS
    size_b = lib.kairo_vocab_loss_backward_workspace_size
    assert size_b(some, 8, 3, 5, 8, some, 8, some, 8, ctypes.byref(n)) == _lib.SUCCESS and n.value >= 256
    assert size_b(some, 8, -3, 5, 8, some, 8, some, 8, ctypes.byref(n)) == _lib.INVALID_VALUE
    assert size_b(some, 8, 3, 5, 8, some, 8, some, 8, None) == _lib.INVALID_VALUE


def test_backward_workspace_follows_the_results():
    """Rows at odd addresses need room for a copy, results that are not wanted none."""
    lib = _lib.lib()

    def size(w=(16, 1000), dx=(16, 1000), dw=(16, 1000)):
        n = ctypes.c_size_t(0)
        assert lib.kairo_vocab_loss_backward_workspace_size(w[0], w[1], 300, 32_000, 1000, dx[0], dx[1], dw[0], dw[1],
                                                            ctypes.byref(n)) == _lib.SUCCESS
        return n.value

    base = size()
    table = 32_000 * 1024 * 2
    assert size(w=(16, 1001)) - base >= table and size(w=(18, 1000)) - base >= table
    assert size(dw=(18, 1000)) - base >= table
    assert size(dw=(None, 1000)) <= base and size(dx=(None, 1000)) <= base


def matrix(blocks=3, b=16, dtype=BF16, rows=32, cols=48):
    nbr = -(-rows // b)
    row_ptr = torch.zeros(nbr + 1, dtype=torch.int32)
    row_ptr[1:] = blocks
    return BlockSparseMatrix(row_ptr=row_ptr, col_idx=torch.arange(blocks, dtype=torch.int32) % 3,
                             blocks=torch.zeros(blocks, b, b, dtype=dtype), shape=(rows, cols), block_size=(b, b))


def host_weights(**kw):
    parts = dict(blocks=torch.zeros(2, 16, 16, dtype=BF16), gate_blocks=1, shape=(16, 32), block=16,
                 ent_ptr=torch.tensor([0, 2], dtype=torch.int32),
                 entries=torch.tensor([[0, 0, -1, 0], [1, -1, 1, 0]], dtype=torch.int32),
                 row_ptr=torch.tensor([0, 1, 2], dtype=torch.int32), col_idx=torch.tensor([0, 1], dtype=torch.int32),
                 blk_idx=torch.tensor([0, 1], dtype=torch.int32), stored_col=torch.tensor([0, 1], dtype=torch.int32))
    return GatedWeights(**{**parts, **kw})


def test_gated_needs_cuda_tensors():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        gated_weights(matrix(), matrix())
    w = host_weights()
    x = torch.zeros(3, 32, dtype=BF16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        sparse_gated_linear(x, w)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        sparse_gated_linear_backward(torch.zeros(3, 16, dtype=BF16), x, w)


def test_gated_arguments():
    w = host_weights()
    assert w.split(w.blocks)[0].shape[0] == 1 and w.with_blocks(w.blocks + 1).blocks[0, 0, 0] == 1
    with pytest.raises(ValueError):
        host_weights(blocks=torch.zeros(3, 16, 16, dtype=BF16))
    with pytest.raises(ValueError):
        host_weights(blocks=torch.zeros(2, 16, 32, dtype=BF16)[:, :, ::2])
    with pytest.raises(ValueError, match="16-byte aligned"):
        host_weights(blocks=torch.zeros(2 * 256 + 1, dtype=BF16)[1:].view(2, 16, 16))
    with pytest.raises(TypeError):
        host_weights(blocks=torch.zeros(2, 16, 16))
    x = torch.zeros(3, 32, dtype=BF16)
    assert gated_module._input("op", x, w, "relu")[1] == 3
    for bad in (x[0], x[:, :31], x.view(1, 3, 32)):
        with pytest.raises(ValueError):
            gated_module._input("op", bad, w, "silu")
    with pytest.raises(ValueError, match="activation"):
        gated_module._input("op", x, w, "tanh")
    with pytest.raises(TypeError):
        gated_module._input("op", x.half(), w, "silu")


def test_gated_c_refusals():
    lib = _lib.lib()
    some, odd = ctypes.c_void_p(256), ctypes.c_void_p(258)

    def desc(rows=100, cols=96, entries=5, blocks=6, b=32, dt=_lib.DTYPE_BF16, ptr=256, ent=256, data=256):
        d = _lib.KairoGated()
        d.rows, d.cols, d.nentries, d.nblocks, d.block, d.dtype = rows, cols, entries, blocks, b, dt
        d.ent_ptr, d.entries, d.blocks = ptr, ent, data
        return d

    def forward(x=some, ldx=96, n=40, act=0, h=some, ldh=100, err=some, **kw):
        return lib.kairo_gated_linear(ctypes.byref(desc(**kw)), x, ldx, n, act, h, ldh, err, None)

    def grad(x=some, ldx=96, n=40, act=0, dh=some, lddh=100, dp=some, lddp=256, err=some, **kw):
        return lib.kairo_gated_linear_grad(ctypes.byref(desc(**kw)), x, ldx, n, act, dh, lddh, dp, lddp, err, None)

    both = ({"x": None}, {"ldx": 95}, {"n": -1}, {"act": 4}, {"act": -1}, {"err": None}, {"rows": -1}, {"entries": -1},
            {"ptr": None}, {"ent": None}, {"data": None}, {"ent": 264}, {"data": 264}, {"x": odd},
            {"ldx": 97})
    for kw in (*both, {"h": None}, {"ldh": 99}):
        assert forward(**kw) == _lib.INVALID_VALUE, kw
        assert lib.kairo_last_error_message()
    for kw in (*both, {"dh": None}, {"dp": None}, {"lddh": 99}, {"lddp": 255}, {"lddp": 260}, {"dp": odd}):
        assert grad(**kw) == _lib.INVALID_VALUE, kw
    for kw in ({"b": 8}, {"b": 128}, {"dt": _lib.DTYPE_F32}, {"n": 1 << 31}, {"blocks": 1 << 30}):
        assert forward(**kw) == _lib.NOT_SUPPORTED, kw
        assert grad(**kw) == _lib.NOT_SUPPORTED, kw
    assert forward(n=0) == _lib.SUCCESS and grad(n=0) == _lib.SUCCESS
    assert lib.kairo_gated_linear(None, some, 96, 4, 0, some, 100, some, None) == _lib.INVALID_VALUE


def test_block_size_and_type_refusals(monkeypatch):
    """The checks of gated_weights behind its device check."""
    class OnDevice(BlockSparseMatrix):
        pass

    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True), raising=False)
    with pytest.raises(ValueError, match="gate is"):
        gated_weights(matrix(rows=32), matrix(rows=48))
    with pytest.raises(TypeError, match="share a dtype"):
        gated_weights(matrix(), matrix(dtype=torch.float16))
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        gated_weights(matrix(dtype=torch.float32), matrix(dtype=torch.float32))
    with pytest.raises(ValueError, match="blocks must be"):
        gated_weights(matrix(b=8), matrix(b=8))


def test_gated_weights_tables():
    """The tables of two patterns on the host: entries, offsets and the stacked order."""
    monkey = pytest.MonkeyPatch()
    monkey.setattr(torch.Tensor, "is_cuda", property(lambda t: True), raising=False)
    try:
        def bsr(rows, cols, perm=None):
            row_ptr = torch.zeros(4, dtype=torch.int32)
            row_ptr[1:] = torch.bincount(torch.tensor(rows), minlength=3).cumsum(0)
            blocks = torch.arange(len(rows), dtype=torch.float32).view(-1, 1, 1).expand(-1, 16, 16).to(BF16).contiguous()
            return BlockSparseMatrix(row_ptr=row_ptr, col_idx=torch.tensor(cols, dtype=torch.int32), blocks=blocks,
                                     shape=(40, 64), block_size=(16, 16),
                                     blk_idx=None if perm is None else torch.tensor(perm, dtype=torch.int32))

        gate, up = bsr([0, 0, 2], [3, 1, 0]), bsr([0, 1, 1, 2], [1, 0, 2, 3], perm=[3, 2, 1, 0])
        w = gated_weights(gate, up)
        assert w.entries.tolist() == [[1, 1, 3, 0], [3, 0, -1, 0], [0, -1, 4, 0], [2, -1, 5, 0], [0, 2, -1, 0],
                                      [3, -1, 6, 0]]
        assert w.ent_ptr.tolist() == [0, 2, 4, 6]
        assert w.row_ptr.tolist() == [0, 2, 3, 3, 5, 6, 7]
        assert w.blk_idx.tolist() == [0, 1, 3, 4, 5, 2, 6] and w.col_idx.tolist() == [3, 1, 1, 0, 2, 0, 3]
        assert w.blocks[:, 0, 0].tolist() == [0, 1, 2, 3, 2, 1, 0]
        with pytest.raises(ValueError, match="twice"):
            gated_weights(bsr([0, 0], [1, 1]), up)
        for bad in (bsr([0], [4]), bsr([0], [-1])):
            with pytest.raises(ValueError, match="malformed"):
                gated_weights(bad, up)
    finally:
        monkey.undo()
