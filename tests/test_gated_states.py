"""Gated projection on the CPU: what its objects keep between calls, and what becomes of it."""

from __future__ import annotations

import pytest
import torch

from kairo_b200 import _lib
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
