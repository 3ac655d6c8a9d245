"""Gated projection: weights whose values, streams, modules or patterns change between calls, against the
same call with weights that were never used before.  Equal inputs give equal bits, so most of it is compared exactly."""

from __future__ import annotations

import copy
import io
from dataclasses import fields, replace

import pytest
import torch

from kairo_b200 import _lib, ops
from kairo_b200.ops import gated as gated_module
from tests.test_gpu_gated import case, weight

pytestmark = pytest.mark.gpu
TYPES = [(torch.bfloat16, torch.float16), (torch.float16, torch.bfloat16)]


def fresh(w):
    """The same weights without anything kept."""
    return replace(w, _structure={})


def step(layer, x, dh):
    """(output, dX, gradients of the parameters) of one training step."""
    for p in layer.parameters():
        p.grad = None
    xr = x.clone().requires_grad_(True)
    y = layer(xr)
    y.backward(dh)
    return [y.detach(), xr.grad, *(p.grad.clone() for p in layer.parameters())]


def same(a, b):
    assert len(a) == len(b)
    for p, q in zip(a, b):
        assert p.dtype == q.dtype and torch.equal(p, q)


@pytest.mark.parametrize("b", [64, 32])
@pytest.mark.parametrize("first,then", TYPES)
def test_values_of_the_other_type(first, then, b):
    """A backward pass in one 16-bit type, then the same patterns with values of the other."""
    x, dh, gate, up, wg, wu = case(300, 200, 136, b, first)
    w = ops.gated_weights(gate, up)
    ops.sparse_gated_linear_backward(dh, x, w, check=True)
    w2, x2, dh2 = w.with_blocks(w.blocks.to(then)), x.to(then), dh.to(then)
    for how in ({}, {"need_dx": False, "dw_dtype": torch.float32}, {"need_dw": False}):
        got = ops.sparse_gated_linear_backward(dh2, x2, w2, check=True, **how)
        want = ops.sparse_gated_linear_backward(dh2, x2, fresh(w2), check=True, **how)
        same([t for t in got if t is not None], [t for t in want if t is not None])
    # and back
    same(ops.sparse_gated_linear_backward(dh, x, w), ops.sparse_gated_linear_backward(dh, x, fresh(w)))


@pytest.mark.parametrize("first,then", TYPES)
def test_module_cast_after_a_step(first, then):
    x, dh, gate, up, wg, wu = case(70, 96, 96, 32, first)
    layer = ops.SparseGatedLinear(gate, up)
    step(layer, x, dh)
    layer.to(then)
    other = ops.SparseGatedLinear(gate, up).to(then)
    same(step(layer, x.to(then), dh.to(then)), step(other, x.to(then), dh.to(then)))


def test_first_backward_on_two_streams(monkeypatch):
    """The kept structure is there before another stream finds it, however long its stream is behind."""
    x, dh, gate, up, wg, wu = case(300, 320, 320, 64, torch.bfloat16)
    w = ops.gated_weights(gate, up)
    want = ops.sparse_gated_linear_backward(dh, x, fresh(w), check=True)
    real = gated_module.bsr_transpose

    def behind(*args, **kw):
        out = real(*args, **kw)
        torch.cuda._sleep(200_000_000)  # what follows on this stream waits about 0.1 s
        return out

    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    monkeypatch.setattr(gated_module, "bsr_transpose", behind)
    with torch.cuda.stream(a):
        got_a = ops.sparse_gated_linear_backward(dh, x, w)
    with torch.cuda.stream(b):
        got_b = ops.sparse_gated_linear_backward(dh, x, w)
    torch.cuda.synchronize()
    same(got_a, want)
    same(got_b, want)


def tensors_of(w):
    return [getattr(w, f.name) for f in fields(w) if isinstance(getattr(w, f.name), torch.Tensor)]


def refill(structure_sizes):
    """Takes memory that was given back on the current stream, and overwrites it with numbers that are no index."""
    return [torch.full((n,), -1, dtype=torch.int32, device="cuda") for n in structure_sizes for _ in range(8)]


def test_structure_freed_while_another_stream_uses_it():
    x, dh, gate, up, wg, wu = case(300, 320, 320, 64, torch.bfloat16)
    w = ops.gated_weights(gate, up)
    want = ops.sparse_gated_linear_backward(dh, x, w, check=True)  # made on this stream
    sizes = [t.numel() for t in w._backward_structure().kept] + [w._backward_structure().perm_stored.numel()]
    b = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(b):
        torch.cuda._sleep(200_000_000)
        got = ops.sparse_gated_linear_backward(dh, x, w)
    for t in tensors_of(w):
        t.record_stream(b)  # the caller's own tensors
    del w
    kept = refill(sizes)
    torch.cuda.synchronize()
    same(got, want)
    del kept


def test_structure_of_a_captured_pass_is_kept():
    """A graph of a training step goes on when its layer's patterns have been loaded again."""
    x, dh, gate, up, wg, wu = case(40, 320, 320, 64, torch.bfloat16)
    layer = ops.SparseGatedLinear(gate, up)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = ops.sparse_gated_linear_backward(dh, x, layer.weights(), check=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = ops.sparse_gated_linear_backward(dh, x, layer.weights())
    st = layer.weights()._backward_structure()
    sizes = [t.numel() for t in st.kept] + [st.perm_stored.numel()]
    del st
    layer.load_state_dict(layer.state_dict())
    with torch.no_grad():
        layer(x)
    kept = refill(sizes)
    g.replay()
    torch.cuda.synchronize()
    same(got, want)
    del kept


def copies(layer):
    """The layer, copied in memory and through a file."""
    buf = io.BytesIO()
    torch.save(layer, buf)
    buf.seek(0)
    return copy.deepcopy(layer), torch.load(buf, weights_only=False)


def test_copies_of_a_trained_module():
    x, dh, gate, up, wg, wu = case(70, 96, 96, 32, torch.bfloat16)
    down, _, _ = weight(96, 96, 32, 0.5, torch.bfloat16, torch.Generator(device="cuda").manual_seed(7))
    for layer in (ops.SparseGatedLinear(gate, up, activation="gelu"), ops.SparseFeedForward(gate, up, down)):
        want = step(layer, x, dh)
        for other in copies(layer):
            same(step(other, x, dh), want)
            with torch.no_grad():
                for p in other.parameters():
                    p.mul_(2)
            twice = step(other, x, dh)
            assert not torch.equal(twice[0], want[0])
            same(step(layer, x, dh), want)  # the copies have tensors of their own


def test_copies_of_weights():
    x, dh, gate, up, wg, wu = case(70, 96, 96, 32, torch.float16)
    w = ops.gated_weights(gate, up)
    want = [ops.sparse_gated_linear(x, w), *ops.sparse_gated_linear_backward(dh, x, w)]
    for other in copies(w):
        assert other.blocks.data_ptr() != w.blocks.data_ptr()
        same([ops.sparse_gated_linear(x, other, check=True), *ops.sparse_gated_linear_backward(dh, x, other, check=True)], want)


def test_layer_made_in_inference_mode():
    x, dh, gate, up, wg, wu = case(40, 96, 96, 32, torch.bfloat16)
    want = [ops.sparse_gated_linear(x, ops.gated_weights(gate, up)),
            *ops.sparse_gated_linear_backward(dh, x, ops.gated_weights(gate, up))]
    with torch.inference_mode():
        layer = ops.SparseGatedLinear(gate, up)
        got = [layer(x), *ops.sparse_gated_linear_backward(dh, x, layer.weights())]
    same(got, want)
    with torch.no_grad():
        same([layer(x)], want[:1])
    # another pattern written over the buffers, whose writes are not counted: nothing is kept from the first
    # (both patterns moved alike, so that they have as many entries together)
    to = torch.tensor([4, 0, 8, 2, 6, 1, 3, 7, 5], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    rows = [torch.repeat_interleave(torch.arange(3, device="cuda"), m.row_ptr.diff().long()) for m in (gate, up)]
    gate2, up2 = (weight(96, 96, 32, 0.4, torch.bfloat16, g, pos=to[r * 3 + m.col_idx.long()])[0]
                  for r, m in zip(rows, (gate, up)))
    with torch.inference_mode():
        other = ops.SparseGatedLinear(gate2, up2)
        layer.load_state_dict(other.state_dict())
        same(ops.sparse_gated_linear_backward(dh, x, layer.weights()),
             ops.sparse_gated_linear_backward(dh, x, other.weights()))


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("table,how", [(1, {"need_dx": False}), (2, {"need_dw": False}), (1, {"need_dw": False})])
def test_errors_of_the_backward_products_can_be_read(table, how, captured):
    """A block-row or position out of range in the kept structure is read nowhere, and recorded where the caller finds it."""
    x, dh, gate, up, wg, wu = case(200, 320, 320, 64, torch.bfloat16)
    w = ops.gated_weights(gate, up)

    def call(check=False):
        return ops.sparse_gated_linear_backward(dh, x, w, check=check, **how)

    call(check=True)
    ops.pending_device_error()
    values = w._backward_structure().kept[table]
    kept = values.clone()
    if captured:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
        values[3] = 1 << 28
        g.replay()
    else:
        values[3] = 1 << 28
        with pytest.raises(_lib.KairoDeviceError) as e:
            call(check=True)
        assert e.value.code & 0xFF == _lib.DEVERR_BAD_INDEX
        call()
    assert ops.pending_device_error() & 0xFF == _lib.DEVERR_BAD_INDEX
    assert ops.pending_device_error() == 0
    values.copy_(kept)
    call(check=True)
    assert ops.pending_device_error() == 0



def test_long_block_column_is_refused():
    """The transposed structure sorts block-columns of up to 16384 stored blocks, gate and up together."""
    rows, b = 8200, 16
    pos = torch.arange(rows, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    gate, wg, _ = weight(rows * b, b, b, 1.0, torch.bfloat16, g, pos=pos)
    up, wu, _ = weight(rows * b, b, b, 1.0, torch.bfloat16, g, pos=pos)
    w = ops.gated_weights(gate, up)
    x = torch.randn(4, b, generator=g, device="cuda").bfloat16()
    h = ops.sparse_gated_linear(x, w, check=True)
    want = torch.nn.functional.silu(x.double() @ wg.t()) * (x.double() @ wu.t())
    assert (h.double() - want).norm() < 2.0**-8 * want.norm()
    for _ in range(2):  # nothing is kept of the refused call
        with pytest.raises(ValueError, match="16384"):
            ops.sparse_gated_linear_backward(h, x, w)


def test_activation_of_the_call():
    """The gradient is that of the function which the forward pass applied."""
    x, dh, gate, up, wg, wu = case(40, 96, 96, 32, torch.bfloat16)
    layer = ops.SparseGatedLinear(gate, up, activation="gelu")
    want = step(layer, x, dh)
    layer.blocks.grad = None
    xr = x.clone().requires_grad_(True)
    h = layer(xr)
    layer.activation = "relu"
    h.backward(dh)
    same([h.detach(), xr.grad, layer.blocks.grad], want)


def test_patterns_of_the_call():
    """Patterns that are replaced or written between the passes change nothing, nor do two forward passes with a writing
    of the same numbers in between."""
    x, dh, gate, up, wg, wu = case(40, 96, 96, 32, torch.bfloat16)
    layer = ops.SparseGatedLinear(gate, up)
    want = step(layer, x, dh)
    layer.blocks.grad = None
    xr = x.clone().requires_grad_(True)
    h = layer(xr)
    kept = layer.col_idx
    layer.col_idx = torch.zeros_like(kept)
    h.backward(dh)
    same([h.detach(), xr.grad, layer.blocks.grad], want)
    layer.col_idx = kept
    buffers = dict(layer.named_buffers())
    before = {k: v.clone() for k, v in buffers.items()}
    for write in (lambda b: b.zero_(), lambda b: b.copy_(b.clone())):
        layer.blocks.grad, xr.grad = None, None
        h = layer(xr)
        for b in buffers.values():
            write(b)
        again = layer(xr)  # of the patterns as they are now
        del again
        h.backward(dh)
        same([h.detach(), xr.grad, layer.blocks.grad], want)
        for k, b in buffers.items():
            b.copy_(before[k])
    same(step(layer, x, dh), want)


def test_passes_of_a_layer_on_two_streams():
    """Forward and backward passes through autograd on two streams at once, the first of a layer among them."""
    x, dh, gate, up, wg, wu = case(300, 320, 320, 64, torch.bfloat16)
    want = step(ops.SparseGatedLinear(gate, up), x, dh)
    layer = ops.SparseGatedLinear(gate, up)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                torch.cuda._sleep(20_000_000)
                xr = x.clone().requires_grad_(True)
                h = layer(xr)
                got.append((h, *torch.autograd.grad(h, (xr, layer.blocks), dh)))
        torch.cuda.synchronize()
        for g in got:
            same(g, want)
        layer.load_state_dict(layer.state_dict())  # the buffers are written again


def test_saved_tensors_that_are_copied():
    x, dh, gate, up, wg, wu = case(40, 96, 96, 32, torch.bfloat16)
    layer = ops.SparseGatedLinear(gate, up)
    want = step(layer, x, dh)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        same(step(layer, x, dh), want)


@pytest.mark.parametrize("tokens", [4, 20, 50, 300, 700])
@pytest.mark.parametrize("b", [64, 32, 16])
def test_malformed_entries_count_as_empty(tokens, b):
    """One bad number of an entry empties all of it, for every token."""
    x, dh, gate, up, wg, wu = case(tokens, 260 * b if tokens == 20 else 3 * b, 4 * b, b, torch.bfloat16, keep=0.9)
    w = ops.gated_weights(gate, up)
    kept = w.entries[1].clone()
    assert (kept[1:3] >= 0).all()  # both weights keep this block
    w.entries[1, 1:3] = -1
    want = ops.sparse_gated_linear(x, w, check=True)
    for field, value in ((0, 4), (0, -1), (1, w.blocks.shape[0]), (2, 1 << 30), (1, -2), (2, -2)):
        w.entries[1] = kept
        w.entries[1, field] = value
        got = ops.sparse_gated_linear(x, w)
        assert ops.pending_device_error() & 0xFF == _lib.DEVERR_BAD_INDEX
        assert torch.equal(got, want)


def test_loaded_patterns_with_another_split():
    """As many blocks in all, of which another number is the gate's."""
    g = torch.Generator(device="cuda").manual_seed(2)
    pos = [torch.tensor(p, device="cuda") for p in ([0, 4, 8], [1, 2, 6], [0, 3, 4, 8], [1, 5])]
    mats = [weight(96, 96, 32, 0.3, torch.bfloat16, g, pos=p)[0] for p in pos]
    one, two = ops.SparseGatedLinear(mats[0], mats[1]), ops.SparseGatedLinear(mats[2], mats[3])
    one.load_state_dict(two.state_dict())
    for w in (one.weights(), copy.deepcopy(one).weights()):
        got, want = w.matrices(), two.weights().matrices()
        for p, q in zip(got, want):
            same([p.row_ptr, p.col_idx, p.blocks], [q.row_ptr, q.col_idx, q.blocks])
        assert [p.shape[0] for p in w.split(w.blocks)] == [4, 2]


def test_layer_loads_without_memory():
    x, dh, gate, up, wg, wu = case(40, 96, 96, 32, torch.bfloat16)
    layer = ops.SparseGatedLinear(gate, up)
    want, bare = step(layer, x, dh), copy.deepcopy(layer).to("meta")
    bare.load_state_dict({k: v.to("meta") for k, v in layer.state_dict().items()})
    bare.load_state_dict(layer.state_dict(), assign=True)
    assert bare.gate_blocks == layer.gate_blocks
    same(step(bare, x, dh), want)


def test_module_refuses_host_tensors():
    x, dh, gate, up, wg, wu = case(8, 64, 64, 32, torch.bfloat16)
    layer = ops.SparseGatedLinear(gate, up)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        layer(x.cpu())
