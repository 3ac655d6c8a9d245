"""Gated projection on the CPU: what its objects keep between calls, and what becomes of it."""

from __future__ import annotations

import copy
import ctypes
import pickle

import pytest
import torch

from kairo_b200 import _lib
from kairo_b200.ops import backward as backward_module
from kairo_b200.ops import gated as gated_module
from kairo_b200.types import BlockSparseMatrix


@pytest.mark.parametrize("then", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("first", [torch.float16, torch.bfloat16])
def test_kept_descriptors_take_the_type_of_the_call(first, then):
    a = BlockSparseMatrix(row_ptr=torch.tensor([0, 1], dtype=torch.int32), col_idx=torch.zeros(1, dtype=torch.int32),
                          blocks=torch.zeros(1, 16, 16, dtype=first), shape=(16, 16), block_size=(16, 16))
    kept = gated_module._bsr_desc(a)
    blocks = torch.zeros(1, 16, 16, dtype=then)
    d = gated_module._with_blocks(kept, blocks)
    assert d.dtype == _lib.kairo_dtype(then) and d.blocks == blocks.data_ptr() and d.nnzb == 1
    assert kept.dtype == _lib.kairo_dtype(first)


def some_weights(dtype=torch.bfloat16):
    i32 = torch.int32
    return gated_module.GatedWeights(
        blocks=torch.arange(512, dtype=torch.float32).view(2, 16, 16).to(dtype), gate_blocks=1, shape=(16, 16), block=16,
        ent_ptr=torch.tensor([0, 1], dtype=i32), entries=torch.tensor([[0, 0, 1, 0]], dtype=i32),
        row_ptr=torch.tensor([0, 1, 2], dtype=i32), col_idx=torch.zeros(2, dtype=i32),
        blk_idx=torch.tensor([0, 1], dtype=i32), stored_col=torch.zeros(2, dtype=i32))


def test_weights_are_copied_without_what_names_their_memory():
    w = some_weights()
    w._structure["backward"] = w._desc  # a descriptor with pointers, as the kept structure has
    for other in (copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        assert other._structure == {} and other.gate_blocks == 1 and other.shape == (16, 16)
        assert torch.equal(other.blocks, w.blocks) and other.blocks.data_ptr() != w.blocks.data_ptr()
        assert other._desc.blocks == other.blocks.data_ptr() and other._desc.entries == other.entries.data_ptr()
    with pytest.raises(AttributeError):
        other.block = 32  # frozen, like the original


def test_error_words_of_the_library():
    n, at = ctypes.c_int32(0), ctypes.c_void_p(None)
    assert _lib.lib().kairo_error_words(None, ctypes.byref(n)) == _lib.INVALID_VALUE
    assert _lib.lib().kairo_error_words(ctypes.byref(at), None) == _lib.INVALID_VALUE


def test_collect_errors_refusals():
    some, lib = ctypes.c_void_p(256), _lib.lib()  # never read: each call is refused first
    two = (ctypes.c_void_p * 2)(256, 256)
    assert lib.kairo_collect_errors(two, 0, some, None) == _lib.INVALID_VALUE
    assert lib.kairo_collect_errors(two, 5, some, None) == _lib.INVALID_VALUE
    assert lib.kairo_collect_errors(two, 2, None, None) == _lib.INVALID_VALUE
    assert lib.kairo_collect_errors(None, 1, some, None) == _lib.INVALID_VALUE
    assert lib.kairo_collect_errors((ctypes.c_void_p * 2)(256, None), 2, some, None) == _lib.INVALID_VALUE


def test_weight_gradient_needs_its_error_word():
    some, d = ctypes.c_void_p(256), _lib.KairoBsr(rows=64, cols=64, bm=64, bk=64, nbr=1, nnzb=0, dtype=_lib.DTYPE_BF16)

    def call(word):
        return _lib.lib().kairo_bsr_sddmm_word(ctypes.byref(d), some, some, some, some, 64, some, 64, 8, some,
                                               _lib.DTYPE_F32, some, 1 << 20, word, None)

    assert call(None) == _lib.INVALID_VALUE and call(some) == _lib.SUCCESS  # no blocks: nothing is launched


def test_entries_without_blocks_are_refused():
    """Every number of the entries is then -1 or out of range; the kernels would copy zeros from behind a block that is not there."""
    lib, some = _lib.lib(), ctypes.c_void_p(256)  # never read: each call is refused first
    w = _lib.KairoGated(rows=64, cols=64, nentries=1, nblocks=0, ent_ptr=256, entries=256, blocks=256, block=64,
                        dtype=_lib.DTYPE_BF16)
    for n in (1, 40, 100, 300):
        assert lib.kairo_gated_linear(ctypes.byref(w), some, 64, n, 0, some, 64, some, None) == _lib.INVALID_VALUE
        assert b"without a stored block" in lib.kairo_last_error_message()
        assert lib.kairo_gated_linear_grad(ctypes.byref(w), some, 64, n, 0, some, 64, some, 128, some,
                                           None) == _lib.INVALID_VALUE
        assert b"without a stored block" in lib.kairo_last_error_message()


def bsr(dtype, n=2, b=16):
    i32 = torch.int32
    return BlockSparseMatrix(row_ptr=torch.tensor([0, n], dtype=i32), col_idx=torch.arange(n, dtype=i32),
                             blocks=torch.zeros(n, b, b, dtype=dtype), shape=(b, n * b), block_size=(b, b))


def test_transposed_values_of_another_type_are_refused():
    t = backward_module.TransposedBsr(matrix=bsr(torch.bfloat16), perm=torch.arange(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="transpose_values"):
        backward_module.transpose_values(bsr(torch.float32), t)
    with pytest.raises(ValueError, match="transpose_values"):
        backward_module.transpose_values(bsr(torch.bfloat16, n=3), t)
    with pytest.raises(ValueError, match="transpose_values"):
        backward_module.transpose_values(bsr(torch.bfloat16, b=32), t)


def test_layer_makes_its_transposed_structure_again_for_another_type(monkeypatch):
    made = []

    def fake(a):
        made.append(a.dtype)
        return backward_module.TransposedBsr(matrix=a, perm=torch.arange(a.nnzb, dtype=torch.int32))

    monkeypatch.setattr(backward_module, "bsr_transpose", fake)
    layer = backward_module.BlockSparseLinear(bsr(torch.bfloat16))
    kept = layer.blocks.detach().clone()
    assert layer.transposed() is layer.transposed() and made == [torch.bfloat16]
    layer.float()
    assert layer.transposed() is layer.transposed() and made[1:] == [torch.float32]
    assert layer.transposed(kept).matrix.dtype == torch.bfloat16  # a pass that began before the cast


def test_layer_loads_without_memory():
    """A layer on the meta device has no pattern to compare."""
    layer = backward_module.BlockSparseLinear(bsr(torch.bfloat16))
    state = layer.state_dict()
    bare = copy.deepcopy(layer).to("meta")
    bare.load_state_dict(state, assign=True)
    assert torch.equal(bare.col_idx, layer.col_idx) and not bare.blocks.is_meta


def test_capture_id_refusals():
    assert _lib.lib().kairo_capture_id(None, None) == _lib.INVALID_VALUE
