"""Workspaces of captured SpMM launches: a graph has its own, whatever eager calls and other graphs do."""

from __future__ import annotations

import pytest
import torch

from kairo_b200 import _lib, ops
from kairo_b200.ops import KernelConfig, block_sparse_mm_bsr
from tests.test_gpu_gated import weight

pytestmark = pytest.mark.gpu


def split_rows(m=512, k=4096, n=256, b=32, seed=0):
    """An SpMM whose long rows are cut between CTAs, which meet at counters and partial sums of the workspace."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    a, dense, _ = weight(m, k, b, 0.4, torch.bfloat16, g)
    cfg = KernelConfig(schedule="rows", num_ctas=100)
    return a, cfg, [torch.randn(k, n, generator=g, device="cuda").bfloat16() for _ in range(2)]


def capture(fn, stream):
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        fn()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out = fn()
    return g, out


def test_graphs_of_one_stream_replay_at_once():
    a, cfg, bs = split_rows()
    want = [block_sparse_mm_bsr(a, b, config=cfg, check=True) for b in bs]
    side = torch.cuda.Stream()

    def calls(b):
        return [block_sparse_mm_bsr(a, b, config=cfg) for _ in range(4)]

    made = [capture(lambda b=b: calls(b), side) for b in bs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for (g, out), s in zip(made, streams):
            for o in out:
                o.fill_(float("nan"))
        torch.cuda.synchronize()
        for (g, out), s in zip(made, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(side):  # beside eager calls on the stream of the captures
            eager = [block_sparse_mm_bsr(a, b, config=cfg) for b in bs]
        torch.cuda.synchronize()
        for (g, out), w, e in zip(made, want, eager):
            assert all(torch.equal(o, w) for o in out) and torch.equal(e, w)


def test_graph_survives_a_larger_eager_workspace():
    a, cfg, bs = split_rows()
    want = block_sparse_mm_bsr(a, bs[0], config=cfg)
    s = torch.cuda.Stream()
    g, out = capture(lambda: block_sparse_mm_bsr(a, bs[0], config=cfg), s)
    with torch.cuda.stream(s):
        before = _lib.workspace(0, torch.device("cuda"))
        size = before.numel()
        after = _lib.workspace(2 * size + 1, torch.device("cuda"))
    assert after.data_ptr() != before.data_ptr()
    del before
    with torch.cuda.stream(s):
        kept = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert all((t == 255).all() for t in kept)


def test_first_call_on_a_stream_in_a_capture():
    a, cfg, bs = split_rows()
    want = block_sparse_mm_bsr(a, bs[0], config=cfg)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        small = ops.sparse_linear(bs[0].t().contiguous(), a)  # another layout and size before it, in one buffer
        out = block_sparse_mm_bsr(a, bs[0], config=cfg)
        again = block_sparse_mm_bsr(a, bs[0], config=cfg)
    for _ in range(3):
        out.zero_(), again.zero_(), small.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(again, want)
        assert torch.equal(small, ops.sparse_linear(bs[0].t().contiguous(), a))


def test_a_replayed_launch_reports_its_error():
    a, cfg, bs = split_rows()
    g, out = capture(lambda: block_sparse_mm_bsr(a, bs[0], config=cfg), torch.cuda.Stream())
    ops.pending_device_error()
    kept = a.col_idx.clone()
    a.col_idx[2] = 1 << 20
    g.replay()
    assert ops.pending_device_error() & 0xFF == _lib.DEVERR_BAD_INDEX
    assert ops.pending_device_error() == 0
    a.col_idx.copy_(kept)
    g.replay()
    assert ops.pending_device_error() == 0


def test_feed_forward_block_in_two_graphs():
    g = torch.Generator(device="cuda").manual_seed(1)
    mats = [weight(m, k, 64, 0.5, torch.bfloat16, g)[0] for m, k in ((1024, 512), (1024, 512), (512, 1024))]
    layer = ops.SparseFeedForward(*mats)
    xs = [torch.randn(300, 512, generator=g, device="cuda").bfloat16() for _ in range(2)]
    side = torch.cuda.Stream()
    with torch.no_grad():
        want = [layer(x) for x in xs]
        made = [capture(lambda x=x: layer(x), side) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for (gr, out), s in zip(made, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, w) for (_, out), w in zip(made, want))


def test_model_step_as_graphed_callables():
    """Forward and backward pass of a feed-forward block and the loss as two graphs that share a pool."""
    g = torch.Generator(device="cuda").manual_seed(1)
    mats = [weight(m, k, 64, 0.5, torch.bfloat16, g)[0] for m, k in ((512, 256), (512, 256), (256, 512))]

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.ffn = ops.SparseFeedForward(*mats)
            self.head = ops.LinearCrossEntropy(torch.nn.Parameter(
                (torch.randn(1000, 256, generator=g, device="cuda") / 16).bfloat16()))

        def forward(self, x, ids):
            return self.head(x + self.ffn(x), ids)

    model = Model()
    xs = [torch.randn(300, 256, generator=g, device="cuda").bfloat16() for _ in range(2)]
    ids = torch.randint(0, 1000, (300,), generator=g, device="cuda")

    def step(f, x):
        xr = x.clone().requires_grad_(True)
        loss = f(xr, ids)
        return [loss.detach().clone(), *(t.clone() for t in torch.autograd.grad(loss, (xr, *model.parameters())))]

    want = [step(model, x) for x in xs]
    graphed = torch.cuda.make_graphed_callables(model, (xs[0].clone().requires_grad_(True), ids.clone()))
    for _ in range(3):
        for x, w in zip(xs, want):
            assert all(torch.equal(a, b) for a, b in zip(step(graphed, x), w))
    assert ops.pending_device_error() == 0
