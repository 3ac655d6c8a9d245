"""Operators called from threads that have made no other CUDA call, autograd's among them."""

from __future__ import annotations

import threading

import pytest
import torch

from kairo_b200 import ops
from tests.test_gpu_gated import case

pytestmark = pytest.mark.gpu


def in_a_thread(call):
    """The call's result, or its error, from a thread of its own."""
    got = {}

    def run():
        try:
            got["value"] = call()
        except Exception as e:  # noqa: BLE001 - raised again below
            got["error"] = e

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if "error" in got:
        raise got["error"]
    return got["value"]


def same(a, b):
    for p, q in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, tuple) else (b,)):
        assert torch.equal(p, q)


def calls():
    x, dh, gate, up, wg, wu = case(300, 192, 256, 64, torch.bfloat16)
    w = ops.gated_weights(gate, up)
    table = torch.randn(1000, 256, device="cuda").bfloat16()
    ids = torch.randint(0, 1000, (300,), device="cuda")
    one = torch.ones((), device="cuda")
    _, lse = ops.linear_cross_entropy(x, table, ids, return_lse=True)
    return {
        "gated, 300 tokens": lambda: ops.sparse_gated_linear(x, w),
        "gated, 50 tokens": lambda: ops.sparse_gated_linear(x[:50], w),
        "gated backward": lambda: ops.sparse_gated_linear_backward(dh, x, w),
        "loss": lambda: ops.linear_cross_entropy(x, table, ids, return_lse=True),
        "loss of few": lambda: ops.linear_cross_entropy(x[:20], table, ids[:20], return_lse=True),
        "loss backward": lambda: ops.linear_cross_entropy_backward(one, x, table, ids, lse),
        "layer": lambda: ops.sparse_linear(x, gate),
    }


@pytest.mark.parametrize("name", ["gated, 300 tokens", "gated, 50 tokens", "gated backward", "loss", "loss of few",
                                  "loss backward", "layer"])
def test_first_call_of_a_thread(name):
    call = calls()[name]
    want = call()
    call()  # what it takes from the allocator has been given back
    torch.cuda.synchronize()
    same(in_a_thread(call), want)


@pytest.mark.parametrize("tokens", [40, 70, 300])
def test_backward_that_autograd_starts_with(tokens):
    """The gradient by a sum is a broadcast number: the projection's backward pass launches first."""
    x, dh, gate, up, wg, wu = case(tokens, 96, 96, 32, torch.bfloat16)
    layer = ops.SparseGatedLinear(gate, up)
    xr = x.clone().requires_grad_(True)
    in_a_thread(lambda: layer(xr).sum().backward())
    dx, db = ops.sparse_gated_linear_backward(torch.ones_like(dh), x, layer.weights(), check=True)
    same((xr.grad, layer.blocks.grad), (dx, db))
