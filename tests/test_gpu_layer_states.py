"""Block-sparse layers whose values or patterns change between training steps, against layers that were never used
before.  Equal inputs give equal bits."""

from __future__ import annotations

import pytest
import torch

from kairo_b200 import ops
from tests.test_gpu_gated import case, weight
from tests.test_gpu_gated_states import same, step

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]  # the types of the layer


def layers(first, b=32, seed=7):
    x, dh, gate, up, wg, wu = case(70, 96, 96, b, first, seed=seed)
    down, _, _ = weight(96, 96, b, 0.5, first, torch.Generator(device="cuda").manual_seed(seed), shuffle=True)
    return x, dh, gate, up, down


@pytest.mark.parametrize("first,then", [(p, q) for p in TYPES for q in TYPES if p != q])
def test_layer_cast_after_a_step(first, then):
    x, dh, gate, up, down = layers(torch.bfloat16)
    x, dh = x.to(first), dh.to(first)
    layer = ops.BlockSparseLinear(down).to(first)
    step(layer, x, dh)
    layer.to(then)
    other = ops.BlockSparseLinear(down).to(first).to(then)
    same(step(layer, x.to(then), dh.to(then)), step(other, x.to(then), dh.to(then)))


@pytest.mark.parametrize("first,then", [(TYPES[0], TYPES[1]), (TYPES[1], TYPES[0])])
def test_feed_forward_cast_after_a_step(first, then):
    x, dh, gate, up, down = layers(first)
    layer = ops.SparseFeedForward(gate, up, down)
    step(layer, x, dh)
    layer.to(then)
    other = ops.SparseFeedForward(gate, up, down).to(then)
    same(step(layer, x.to(then), dh.to(then)), step(other, x.to(then), dh.to(then)))


def test_adapted_layer_cast_after_a_step():
    x, dh, gate, up, down = layers(torch.bfloat16)
    plan = ops.adapter_plan(torch.zeros(70, dtype=torch.int32, device="cuda"), 1)
    one, two = (ops.AdaptedSparseLinear(ops.BlockSparseLinear(down), 1, 8) for _ in range(2))
    two.load_state_dict(one.state_dict())

    def grads(layer, x, dh):
        for p in layer.parameters():
            p.grad = None
        xr = x.clone().requires_grad_(True)
        layer(xr, plan).backward(dh)
        return [xr.grad, *(p.grad for p in layer.parameters())]

    grads(one, x, dh)
    same(grads(one.half(), x.half(), dh.half()), grads(two.half(), x.half(), dh.half()))


@pytest.mark.parametrize("b", [64, 32])
def test_loaded_patterns_are_followed(b):
    """A state dict of another pattern with as many blocks, after a step: a layer alone and in a feed-forward block."""
    g = torch.Generator(device="cuda").manual_seed(1)
    n = 3 * b
    mats = [weight(n, n, b, 0.3, torch.bfloat16, g, pos=torch.tensor(p, device="cuda"))[0]
            for p in ([0, 1, 2], [0, 4, 7], [2, 3, 8])]
    x, dh = torch.randn(70, n, device="cuda").bfloat16(), torch.randn(70, n, device="cuda").bfloat16()
    for make in (lambda m: ops.BlockSparseLinear(m), lambda m: ops.SparseFeedForward(mats[2], mats[2], m)):
        one, two = make(mats[0]), make(mats[1])
        step(one, x, dh)
        one.load_state_dict(two.state_dict())
        same(step(one, x, dh), step(two, x, dh))
        layer = one if isinstance(one, ops.BlockSparseLinear) else one.down
        assert layer.max_row_blocks == mats[1].max_row_blocks
        kept = layer.transposed()
        one.load_state_dict(two.state_dict())
        assert layer.transposed() is kept  # the same pattern: the structure stays, as captured graphs expect


def test_structure_of_a_captured_step_is_kept():
    """A graph of a backward pass replays with the structure that it was captured with, after another pattern was loaded."""
    g = torch.Generator(device="cuda").manual_seed(3)
    one, two = (ops.BlockSparseLinear(weight(192, 192, 64, 0.3, torch.bfloat16, g, pos=torch.tensor(p, device="cuda"))[0])
                for p in ([0, 1, 2, 5], [0, 4, 7, 8]))
    dy, x = torch.randn(70, 192, device="cuda").bfloat16(), torch.randn(70, 192, device="cuda").bfloat16()
    W, blocks = one.weight_matrix(), one.blocks.detach().clone()

    def grads():
        return ops.sparse_linear_backward(dy, x, W, ops.transpose_values(W, one.transposed()))

    want = [t.clone() for t in grads()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = grads()
    sizes = [t.numel() for t in (one.transposed().matrix.row_ptr, one.transposed().matrix.col_idx, one.transposed().perm)]
    pattern = one.row_ptr.clone(), one.col_idx.clone()
    one.load_state_dict(two.state_dict())
    kept = [torch.full((n,), -1, dtype=torch.int32, device="cuda") for n in sizes for _ in range(8)]
    with torch.no_grad():
        one.blocks.copy_(blocks)
        one.row_ptr.copy_(pattern[0])
        one.col_idx.copy_(pattern[1])
    graph.replay()
    torch.cuda.synchronize()
    same(got, want)
    del kept
