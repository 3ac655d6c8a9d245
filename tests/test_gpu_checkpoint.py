"""Activations in 8 bits, and the weight gradient taken from them.

Codes and steps are defined by a few fp32 operations and one rounding of an
exact product, so they are compared bit for bit with the same definition in
64 bits.  The weight gradient is compared with the 64-bit product of dY and
the activation as it reads back: n fp32 (or tensor-core, truncating) additions
are off by at most n * 2^-23 of the sum of magnitudes, plus half a step of the
output.
"""

from __future__ import annotations

import pytest
import torch

from kairo_b200.ops import (
    BlockSparseLinear,
    QuantizedActivations,
    bsr_from_tiles,
    bsr_transpose,
    dequantize_activations,
    quantize_activations,
    sparse_linear_backward,
    sparse_linear_weight_grad,
)

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _define(x):
    """codes (n, k) int8, steps (g, n) and the activation read back, by the definition."""
    n, k = x.shape
    groups = (k + 63) // 64
    xf = torch.zeros(n, groups * 64, dtype=torch.float64)
    xf[:, :k] = x.double().cpu()
    xf = xf.view(n, groups, 64)
    finite = xf.isfinite().all(2)
    a = torch.where(finite, xf.abs().amax(2), 1.0).float()
    live = finite & (a >= 2.0**-100)
    inv = torch.where(live, a.reciprocal() * 127.0, 0.0)
    codes = (torch.where(live[..., None], xf, 0.0) * inv[..., None].double()).round().to(torch.int8)
    steps = torch.where(live, a * torch.tensor(1.0 / 127.0, dtype=torch.float32), torch.where(finite, 0.0, float("nan")))
    back = (codes.float() * steps[..., None]).view(n, -1)[:, :k].to(x.dtype)
    return codes.view(n, -1)[:, :k], steps.t(), back


def _same(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def _check(x):
    codes, steps, back = _define(x)
    q = quantize_activations(x)
    assert torch.equal(q.codes.cpu(), codes)
    assert _same(q.steps.cpu(), steps)
    y = dequantize_activations(q)
    assert y.dtype == x.dtype and _same(y.cpu(), back)
    return q, back


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 64), (3, 65), (7, 127), (33, 256), (31, 257), (100, 1000), (257, 777)])
def test_round_trip(dt, shape):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(shape[1])).to(dt)
    x[:, ::50] *= 30
    if shape[0] > 2:
        x[1] = 0
    q, back = _check(x.to(DEV))
    # half a step of the code, and half a step of the type
    half = torch.finfo(dt).eps / 2
    groups = torch.nn.functional.pad(x.double(), (0, -shape[1] % 64)).view(shape[0], -1, 64)
    a = groups.abs().amax(2, keepdim=True).expand_as(groups).reshape(shape[0], -1)[:, : shape[1]]
    assert bool(((back.double() - x.double()).abs() <= a / 254 * (1 + 2.0**-20) + a * half * 1.01).all())


def test_ties_and_extremes():
    x = torch.zeros(8, 64)
    x[0] = torch.arange(64) / 2.0 - 16        # halves: ties to even under a power-of-two step ...
    x[0, 0] = 127.0                           # ... (step 1)
    x[1] = torch.linspace(-1, 1, 64) * torch.finfo(torch.float32).max
    x[2] = torch.linspace(-1, 1, 64) * 2.0**-99.5
    x[3] = torch.linspace(-1, 1, 64) * 2.0**-101
    x[4, 5] = 2.0**-149
    x[5] = -0.0
    x[6, 3] = float("inf")
    x[7, 9] = float("nan")
    q, back = _check(x.to(DEV))
    assert q.codes[0, 1:4].tolist() == [-16, -15, -14]  # -15.5, -15, -14.5
    assert bool((back[3] == 0).all()) and bool(back[6].isnan().all()) and bool(back[7].isnan().all())
    h = torch.tensor([[65504.0, -65504.0, 6e-8, 1.0]], dtype=torch.float16)
    _check(h.to(DEV))
    _check(torch.full((1, 70), 6e-8, dtype=torch.float16, device=DEV))  # fp16 subnormals keep their codes


@pytest.mark.parametrize("dt", TYPES)
def test_strides(dt):
    wide = torch.randn(40, 400, device=DEV).to(dt)
    for view in (wide[:, 8:136], wide[:, 3:200], wide[::3, :130], wide.t(), wide[:1].expand(5, 400)):
        _check(view)
    q = quantize_activations(wide[:, :100])
    out = torch.full((41, 120), 7.0, dtype=dt, device=DEV)
    dequantize_activations(q, out=out[:40, :100])
    assert _same(out[:40, :100].cpu(), _define(wide[:, :100])[2])
    assert bool((out[40] == 7).all()) and bool((out[:, 100:] == 7).all())
    assert quantize_activations(wide[:0]).shape == (0, 400)
    assert dequantize_activations(quantize_activations(wide[:, :0])).shape == (40, 0)
    # codes inside a wider buffer of the caller's
    buf = torch.full((40, 256), 9, dtype=torch.int8, device=DEV)
    inner = QuantizedActivations(codes=buf[:, 16:116], steps=q.steps, dtype=dt)
    inner.codes.copy_(q.codes)
    assert torch.equal(dequantize_activations(inner), dequantize_activations(q))


def test_offsets_pass_32_bits():
    x = torch.zeros(70_000, 32_768, dtype=torch.bfloat16, device=DEV)
    x[-1, -1], x[-1, -64], x[-2, 7] = 3.0, -3.0, 5.0
    q = quantize_activations(x)
    assert q.codes[-1, -1].item() == 127 and q.codes[-1, -64].item() == -127 and q.codes[-2, 7].item() == 127
    assert torch.equal(dequantize_activations(q), x)


def _layer(dt, m, k, bs, keep, seed):
    g = torch.Generator().manual_seed(seed)
    nbr, nbc = -(-m // bs), -(-k // bs)
    pos = torch.sort(torch.randperm(nbr * nbc, generator=g)[:max(1, int(nbr * nbc * keep))]).values
    tiles = (torch.randn(pos.numel(), bs, bs, generator=g) * 0.1).to(dt)
    return bsr_from_tiles(tiles.to(DEV), (pos // nbc).int().to(DEV), (pos % nbc).int().to(DEV), (m, k)), pos


def _grad_ref(dy, back, m, k, bs, pos):
    nbr, nbc = -(-m // bs), -(-k // bs)

    def full(a, b):
        d = torch.zeros(nbr * bs, nbc * bs, dtype=torch.float64, device=DEV)
        d[:m, :k] = a.t() @ b
        return d.view(nbr, bs, nbc, bs).permute(0, 2, 1, 3).reshape(-1, bs, bs)[pos.to(DEV)]

    a, b = dy.double().to(DEV), back.double().to(DEV)
    return full(a, b), full(a.abs(), b.abs())


@pytest.mark.parametrize("case", [
    # dtype, out, batch, m, k, block, keep
    (torch.bfloat16, torch.float32, 200, 512, 640, 64, 0.3),
    (torch.bfloat16, torch.bfloat16, 1, 256, 256, 64, 0.5),
    (torch.float16, torch.float16, 64, 128, 1024, 64, 1.0),
    (torch.float16, torch.float32, 333, 300, 200, 64, 0.7),     # ragged: edges inside a block and a group
    (torch.bfloat16, torch.float32, 65, 264, 1000, 64, 0.4),
    (torch.bfloat16, torch.float32, 777, 4096, 64, 64, 1.0),    # one long block-column
    (torch.float16, torch.float32, 90, 128, 192, 32, 0.5),
    (torch.bfloat16, torch.bfloat16, 50, 96, 80, 16, 0.5),
    (torch.float32, torch.float32, 70, 128, 96, 32, 0.5),
])
def test_weight_grad(case):
    dt, ot, n, m, k, bs, keep = case
    w, pos = _layer(dt, m, k, bs, keep, seed=n)
    g = torch.Generator().manual_seed(n + 1)
    x = torch.randn(n, k, generator=g).to(dt).to(DEV)
    x[:, ::37] *= 20
    dy = (torch.randn(n, m, generator=g) * 0.1).to(dt).to(DEV)
    q = quantize_activations(x)
    back = _define(x)[2]
    ref, mag = _grad_ref(dy, back, m, k, bs, pos)
    half = torch.finfo(ot).eps / 2
    for wt in (None, bsr_transpose(w)):
        dw = sparse_linear_weight_grad(dy, q, w, wt, out_dtype=ot, check=True)
        err = (dw.double() - ref).abs()
        tol = mag * n * 2.0**-23 + ref.abs() * half * 1.01 + torch.finfo(ot).smallest_normal * half * 2
        assert bool((err <= tol).all())
    # dX is the forward kernel's: 16-bit types, 16-byte rows of dY
    dx, dw2 = sparse_linear_backward(dy, q, w, need_dx=dt != torch.float32 and m % 8 == 0, dw_dtype=ot)
    assert torch.equal(dw, dw2) and (dx is None or dx.dtype == dt)


def test_weight_grad_edges():
    w, pos = _layer(torch.bfloat16, 256, 256, 64, 0.5, seed=1)
    x = torch.randn(0, 256, device=DEV, dtype=torch.bfloat16)
    assert bool((sparse_linear_weight_grad(x, quantize_activations(x), w) == 0).all())  # no rows in the batch
    x = torch.randn(100, 256, device=DEV, dtype=torch.bfloat16)
    q = quantize_activations(x)
    wide = torch.randn(100, 600, device=DEV, dtype=torch.bfloat16)
    for dy in (wide[:, 8:264], wide[:, 3:259]):  # 16-byte rows and unaligned ones
        ref, mag = _grad_ref(dy, _define(x)[2], 256, 256, 64, pos)
        dw = sparse_linear_weight_grad(dy, q, w)
        assert bool(((dw.double() - ref).abs() <= mag * 100 * 2.0**-23 + ref.abs() * 2.0**-24).all())
    with pytest.raises(TypeError):
        sparse_linear_weight_grad(wide[:, :256], quantize_activations(x.half()), w)
    with pytest.raises(ValueError):
        sparse_linear_weight_grad(wide[:, :256], quantize_activations(x[:50]), w)
    x[7, 70] = float("nan")  # stays visible in the blocks of its column group, and nowhere else
    dw = sparse_linear_weight_grad(wide[:, :256].contiguous(), quantize_activations(x), w)
    hit = (pos % 4 == 1).to(DEV)
    assert bool(dw[hit].isnan().all()) and bool(dw[~hit].isfinite().all())


def test_module_keeps_its_input_in_8_bits():
    w, pos = _layer(torch.bfloat16, 256, 512, 64, 0.4, seed=5)
    plain, kept = BlockSparseLinear(w), BlockSparseLinear(w, checkpoint="int8")
    x = torch.randn(96, 512, device=DEV, dtype=torch.bfloat16)
    dy = torch.randn(96, 256, device=DEV, dtype=torch.bfloat16) * 0.1
    xs = [x.clone().requires_grad_() for _ in range(2)]
    saved = []

    def pack(t):
        saved.append(t)
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = kept(xs[1])
    assert not any(t.dtype == torch.bfloat16 and t.shape == x.shape for t in saved)
    assert sum(t.numel() * t.element_size() for t in saved if t.shape[0] != w.nnzb) <= x.numel() * (1 + 1 / 16)
    y0 = plain(xs[0])
    assert torch.equal(y, y0)
    y.backward(dy)
    y0.backward(dy)
    assert torch.equal(xs[0].grad, xs[1].grad)  # dX does not depend on the checkpoint
    ref, mag = _grad_ref(dy, _define(x)[2], 256, 512, 64, pos)
    tol = mag * 96 * 2.0**-23 + ref.abs() * 2.0**-8 * 1.01
    assert bool(((kept.blocks.grad.double() - ref).abs() <= tol).all())
    assert not torch.equal(kept.blocks.grad, plain.blocks.grad)
    kept.blocks.requires_grad_(False)  # a frozen layer keeps nothing for dW
    saved.clear()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        kept(xs[1])
    assert not any(t.dtype == torch.int8 or t.shape == x.shape for t in saved)
    xg = x.clone().requires_grad_()
    kept(xg).backward(dy)
    assert torch.equal(xg.grad, xs[0].grad)


def test_out_must_not_share_memory():
    x = torch.randn(8, 64, device=DEV)
    q = quantize_activations(x)
    buf = torch.empty(8 * 64 * 4, dtype=torch.uint8, device=DEV)
    codes = buf[:512].view(torch.int8).view(8, 64)
    codes.copy_(q.codes)
    with pytest.raises(ValueError, match="share memory"):
        dequantize_activations(QuantizedActivations(codes=codes, steps=q.steps, dtype=torch.float32),
                               out=buf.view(torch.float32).view(8, 64))


def test_streams_and_graph():
    w, pos = _layer(torch.bfloat16, 512, 512, 64, 0.3, seed=6)
    wt = bsr_transpose(w)
    x = torch.randn(300, 512, device=DEV, dtype=torch.bfloat16)
    dy = torch.randn(300, 512, device=DEV, dtype=torch.bfloat16)

    def step():
        q = quantize_activations(x)
        return dequantize_activations(q), sparse_linear_weight_grad(dy, q, w, wt)

    ref = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
        graphs.append((g, out))
    x.normal_()
    ref = step()
    for g, out in graphs:
        for t in out:
            t.fill_(float("nan"))
    for _ in range(2):
        for g, _out in graphs:
            g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(ref, out))
