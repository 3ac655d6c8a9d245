"""Corners of the operators around the linear layer on the device.

Plain implementations are in 64 bits.  Tolerances count half steps of the
output's type (torch.finfo(t).eps / 2 of the value) and, for a sum of n products in
fp32, n * 2^-23 of the sum of magnitudes.
"""

from __future__ import annotations

import pytest
import torch

from kairo_b200.ops import (
    BlockSparseLinear,
    LowRankAdapters,
    adapter_linear,
    adapter_plan,
    bsr_from_tiles,
    dequantize_activations,
    quantize_activations,
    sparse_linear_weight_grad,
)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _half(t):
    return torch.finfo(t).eps / 2


def _weight(dt, m, k, bs=64, seed=0):
    """A weight with every second block of a checkerboard, its block-rows and block-columns."""
    nbr, nbc = -(-m // bs), -(-k // bs)
    pos = torch.tensor([p for p in range(nbr * nbc) if (p // nbc + p % nbc) % 2 == 0])
    tiles = (torch.randn(pos.numel(), bs, bs, generator=torch.Generator().manual_seed(seed)) * 0.1).to(dt)
    rows, cols = pos // nbc, pos % nbc
    return bsr_from_tiles(tiles.to(DEV), rows.int().to(DEV), cols.int().to(DEV), (m, k)), rows.to(DEV), cols.to(DEV)


def _blocks(dense, rows, cols, bs=64):
    m, k = dense.shape
    pad = torch.nn.functional.pad(dense, (0, -k % bs, 0, -m % bs))
    return pad.view(-(-m // bs), bs, -(-k // bs), bs).permute(0, 2, 1, 3)[rows, cols]


@pytest.mark.parametrize("bs", [64, 32])
def test_weight_grad_of_a_broadcast_gradient(bs):
    """dY whose rows share or overlap memory is read as the values that it stands for."""
    w, rows, cols = _weight(torch.bfloat16, 128, 192, bs)
    x = torch.randn(300, 192, device=DEV).bfloat16()
    q = quantize_activations(x)
    back = dequantize_activations(q).double()
    one = torch.randn(128, device=DEV).bfloat16()
    long = torch.randn(300 * 8 + 128, device=DEV).bfloat16()
    for dy in (one.expand(300, 128), long.as_strided((300, 128), (8, 1))):
        got = sparse_linear_weight_grad(dy, q, w)
        ref = _blocks(dy.double().t() @ back, rows, cols, bs)
        mag = _blocks(dy.double().abs().t() @ back.abs(), rows, cols, bs)
        assert bool(((got.double() - ref).abs() <= mag * 300 * 2.0**-23 + ref.abs() * 2.0**-24).all())
        assert torch.equal(got, sparse_linear_weight_grad(dy.contiguous(), q, w))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [8192, 8193, (1 << 20) + 77])
def test_weight_grad_of_a_long_batch(dt, n):
    """Values of one sign, where the matrix units' truncation adds up: a 16-bit result stays at its own rounding."""
    w = bsr_from_tiles(torch.zeros(1, 64, 64, dtype=dt, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV),
                       torch.zeros(1, dtype=torch.int32, device=DEV), (64, 64))
    torch.manual_seed(n)
    x = (torch.rand(n, 64, device=DEV) * 0.01 + 0.005).to(dt)
    dy = (torch.rand(n, 64, device=DEV) * 0.01 + 0.005).to(dt)
    q = quantize_activations(x)
    ref = dy.double().t() @ dequantize_activations(q).double()
    # a sum of 8192 rows: 512 steps, each with a truncation inside the units and one of the sum; the sums of
    # up to 129 such segments are added in fp32
    lost = 512 * 2 * 2.0**-23 + 129 * 2.0**-24
    got = sparse_linear_weight_grad(dy, q, w, out_dtype=dt)[0]
    assert bool(((got.double() - ref).abs() <= ref * (lost + _half(dt) * (1 + lost))).all())
    # fp32 results: 48 steps a segment, up to 1367 segments
    lost = 48 * 2 * 2.0**-23 + 1367 * 2.0**-24
    got = sparse_linear_weight_grad(dy, q, w, out_dtype=torch.float32)[0]
    assert bool(((got.double() - ref).abs() <= ref * lost).all())


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", [131072, 131073, (1 << 20) + 8, (1 << 20) + 3])
@pytest.mark.parametrize("rank,t", [(4, 3), (20, 18), (40, 1), (100, 2)])
def test_long_contractions(dt, k, rank, t):
    """fp32 results of features of one sign, on both sides of the length up to which the units keep one sum."""
    gen = torch.Generator(device=DEV).manual_seed(k + rank)
    x = (torch.rand(t, k, generator=gen, device=DEV) + 0.5).to(dt)
    down = ((torch.rand(2, rank, k, generator=gen, device=DEV) + 0.5) * 2**-8).to(dt)
    up = torch.ones(2, rank, 72, dtype=dt, device=DEV)
    ids = torch.arange(t, device=DEV) % 3 - 1  # the last of every three: adapter 1
    plan = adapter_plan(ids, 2)
    y, low = adapter_linear(x, LowRankAdapters(down=down, up=up), plan, out_dtype=torch.float32, return_low=True)
    ref = torch.einsum("tk,trk->tr", x.double(), down.double()[ids.clamp(min=0)]) * (ids >= 0)[:, None]
    # 128 products in a part, each with a truncation inside the units and one of the sum; up to 8 parts, 8 warps and 8 CTAs
    lost = 128 * 2 * 2.0**-23 + 24 * 2.0**-24
    assert bool(((low.double() - ref).abs() <= ref * lost).all())
    want = ref.sum(1, keepdim=True).expand(t, 72)
    assert bool(((y.double() - want).abs() <= want * (lost + (rank + 4) * 2.0**-23)).all())
