"""Low-rank adapters of many requests beside a shared projection.

The plain implementation is in 64 bits.  With |.| the same product of
magnitudes: low is a sum of K products (fp32 additions, truncating on the tensor
cores: 2^-23 each), Y adds R products of it.  Between the two, low may be held
as a few 16-bit terms whose rest is at most 2^-17 of it (16-bit results) or
2^-23 (fp32 results).  Then one rounding to the output's type.
"""

from __future__ import annotations

import pytest
import torch

from kairo_b200 import _lib
from kairo_b200.ops import (
    AdaptedSparseLinear,
    BlockSparseLinear,
    LowRankAdapters,
    ScaledEmbedding,
    adapted_sparse_linear,
    adapter_linear,
    adapter_linear_backward,
    adapter_plan,
    bsr_from_tiles,
    dequantize_activations,
    quantize_activations,
)

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def _rest(t):
    return 2.0**-23 if t == torch.float32 else 2.0**-17


def _round_tol(ref, slack, t):
    half = torch.finfo(t).eps / 2
    return slack + (ref.abs() + slack) * half * 1.01 + torch.finfo(t).smallest_normal * half * 2


def _problem(dt, t, k, n, r, g, seed, order="mixed"):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(t, k, generator=gen).to(dt).to(DEV)
    dy = (torch.randn(t, n, generator=gen) * 0.1).to(dt).to(DEV)
    down = (torch.randn(g, r, k, generator=gen) * k**-0.5).to(dt).to(DEV)
    up = (torch.randn(g, r, n, generator=gen) * r**-0.5).to(dt).to(DEV)
    scale = (0.5 + torch.rand(g, generator=gen)).to(DEV)
    ids = torch.randint(-1, g + 1, (t,), generator=gen)  # -1 and g: none
    if order == "packed":
        ids = torch.sort(ids).values
    return x, dy, LowRankAdapters(down=down, up=up, scale=scale), ids


def _forward(x, a, ids, base, swap=False):
    """Y, low and their magnitudes; with swap the two factors change places (the backward product)."""
    down, up = (a.up, a.down) if swap else (a.down, a.up)
    scale = torch.ones(a.count) if a.scale is None else a.scale
    x, down, up, scale, ids = x.double(), down.double(), up.double(), scale.double().to(x.device), ids.to(x.device)
    y = torch.zeros(x.shape[0], up.shape[2], dtype=torch.float64, device=x.device) if base is None else base.double()
    y, mag = y.clone(), y.abs()
    low = torch.zeros(x.shape[0], a.rank, dtype=torch.float64, device=x.device)
    low_mag = low.clone()
    for i in range(a.count):
        at = (ids == i).nonzero().flatten()
        low[at] = scale[i] * (x[at] @ down[i].t())
        low_mag[at] = scale[i] * (x[at].abs() @ down[i].abs().t())
        y[at] += low[at] @ up[i]
        mag[at] += low_mag[at] @ up[i].abs()
    return y, mag, low, low_mag


def _wgrad(s, s_mag, z, a, ids):
    ids = ids.to(z.device)
    out = torch.zeros(a.count, s.shape[1], z.shape[1], dtype=torch.float64, device=z.device)
    mag = torch.zeros_like(out)
    for i in range(a.count):
        at = (ids == i).nonzero().flatten()
        out[i] = s[at].t() @ z[at].double()
        mag[i] = s_mag[at].t() @ z[at].double().abs()
    return out, mag


def _check(x, dy, a, ids, base, base_dx, out_dtype=None, grad_dtype=None):
    t, k, n, r = x.shape[0], a.in_features, a.out_features, a.rank
    plan = adapter_plan(ids.to(DEV), a.count)
    y, low = adapter_linear(x, a, plan, base=base, out_dtype=out_dtype, return_low=True)
    odt = out_dtype or x.dtype
    assert y.dtype == odt and low.dtype == torch.float32
    ry, my, rl, ml = _forward(x, a, ids, base)
    assert bool(((low.double() - rl).abs() <= ml * (k + 2) * 2.0**-23).all())
    slack = my * ((k + r + 4) * 2.0**-23 + _rest(odt))
    assert bool(((y.double() - ry).abs() <= _round_tol(ry, slack, odt)).all())
    gdt = grad_dtype or x.dtype
    for given in (low, None):
        dx, dd, du = adapter_linear_backward(dy, x, a, plan, low=given, base_dx=base_dx, grad_dtype=grad_dtype)
        rx, mx, rdl, mdl = _forward(dy, a, ids, base_dx, swap=True)
        slack = mx * ((n + r + 4) * 2.0**-23 + _rest(x.dtype))
        assert bool(((dx.double() - rx).abs() <= _round_tol(rx, slack, x.dtype)).all())
        for got, (ref, mag), terms in ((dd, _wgrad(rdl, mdl, x, a, ids), n), (du, _wgrad(rl, ml, dy, a, ids), k)):
            assert got.dtype == gdt
            slack = mag * ((terms + t + 4) * 2.0**-23 + _rest(gdt))
            assert bool(((got.double() - ref).abs() <= _round_tol(ref, slack, gdt)).all())
    return y


CASES = [
    # tokens, in, out, rank, adapters
    (1, 64, 64, 8, 1),
    (1, 2048, 1024, 16, 5),
    (7, 256, 520, 16, 9),
    (40, 1000, 1032, 4, 64),      # more adapters than some tokens use
    (33, 130, 70, 5, 3),          # rows of no 16-byte multiple
    (65, 77, 33, 1, 2),
    (200, 512, 384, 12, 4),
    (300, 640, 768, 64, 3),
    (129, 256, 256, 128, 2),
    (515, 320, 264, 33, 1),
    (2100, 128, 192, 16, 3),      # from here on the tall tiles of long batches
    (2300, 136, 128, 30, 5),
    (2300, 192, 136, 64, 3),
    (2200, 128, 200, 100, 2),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", CASES)
def test_forward_and_backward(dt, case):
    t, k, n, r, g = case
    x, dy, a, ids = _problem(dt, t, k, n, r, g, seed=t + k, order="mixed" if t % 2 else "packed")
    gen = torch.Generator().manual_seed(1)
    base = torch.randn(t, n, generator=gen).to(DEV)
    base_dx = torch.randn(t, k, generator=gen).to(DEV)
    _check(x, dy, a, ids, base.to(dt), base_dx.to(dt))
    _check(x, dy, a, ids, base, base_dx, out_dtype=torch.float32, grad_dtype=torch.float32)
    _check(x, dy, LowRankAdapters(down=a.down, up=a.up), ids.int(), None, None)


def test_batches_and_none():
    x, dy, a, _ = _problem(torch.bfloat16, 50, 128, 256, 8, 4, seed=0)
    base = torch.randn(50, 256, device=DEV).bfloat16()
    for ids in (torch.full((50,), -1), torch.full((50,), 4), torch.full((50,), 2), torch.arange(50) % 4,
                torch.arange(50) - 10):
        y = _check(x, dy, a, ids, base, None)
        none = ((ids < 0) | (ids >= 4)).to(DEV)
        assert torch.equal(y[none], base[none])
    plan = adapter_plan(torch.zeros(0, dtype=torch.int64, device=DEV), 4)
    y, low = adapter_linear(x[:0], a, plan, return_low=True)
    assert y.shape == (0, 256) and low.shape == (0, 8)
    dx, dd, du = adapter_linear_backward(dy[:0], x[:0], a, plan, low=low)
    assert dx.shape == (0, 128) and bool((dd == 0).all()) and bool((du == 0).all())
    none = LowRankAdapters(down=a.down[:0], up=a.up[:0])  # no adapter loaded at all
    plan = adapter_plan(torch.zeros(50, dtype=torch.int64, device=DEV), 0)
    assert torch.equal(adapter_linear(x, none, plan, base=base), base)
    assert bool((adapter_linear(x, none, plan) == 0).all())


@pytest.mark.parametrize("t", [5, 300])
def test_strides_in_place_and_rows_behind(t):
    k, n = 256, 192
    x, dy, a, ids = _problem(torch.bfloat16, t, k, n, 16, 3, seed=t)
    plan = adapter_plan(ids.to(DEV), 3)
    for off, pad in ((8, 24), (3, 7)):  # 16-byte rows, and unaligned ones
        wide_x = torch.randn(t, k + pad, device=DEV).bfloat16()
        xv = wide_x[:, off:off + k] if off + k <= k + pad else wide_x[:, pad:]
        wide_y = torch.randn(t + 2, n + pad, device=DEV).bfloat16()
        before = wide_y.clone()
        yv = wide_y[:t, pad:]
        ref, mag, _, _ = _forward(xv, a, ids, yv)
        got = adapter_linear(xv, a, plan, base=yv, out=yv)
        assert got is yv
        slack = mag * ((k + 20) * 2.0**-23 + 2.0**-17)
        assert bool(((yv.double() - ref).abs() <= _round_tol(ref, slack, torch.bfloat16)).all())
        assert torch.equal(wide_y[t:], before[t:]) and torch.equal(wide_y[:, :pad], before[:, :pad])
    xt = torch.randn(k, t, device=DEV).bfloat16().t()  # columns contiguous
    assert torch.equal(adapter_linear(xt, a, plan), adapter_linear(xt.contiguous(), a, plan))
    assert torch.equal(adapter_linear(x[:1].expand(t, k), a, plan), adapter_linear(x[:1].repeat(t, 1), a, plan))


def test_nonfinite_rows_stay_with_their_tokens():
    x, dy, a, ids = _problem(torch.bfloat16, 48, 128, 64, 8, 3, seed=2)
    ids = torch.arange(48) % 4 - 1
    plan = adapter_plan(ids.to(DEV), 3)
    clean = adapter_linear(x, a, plan)
    x[5, 3], x[8, 9], x[6, 1] = float("inf"), float("nan"), -float("inf")  # tokens of adapters 0, none, 1
    y = adapter_linear(x, a, plan)
    rest = [i for i in range(48) if i not in (5, 6)]
    assert torch.equal(y[rest], clean[rest])
    assert not bool(y[5].isfinite().any()) and not bool(y[6].isfinite().any())
    down = a.down.clone()
    down[2] = float("nan")  # an adapter that is broken spoils only its own tokens
    y = adapter_linear(x, LowRankAdapters(down=down, up=a.up, scale=a.scale), plan)
    other = [i for i in rest if int(ids[i]) != 2]
    assert torch.equal(y[other], clean[other]) and bool(y[(ids == 2).to(DEV)].isnan().all())


def test_small_gradients_in_fp16():
    """dY far under fp16's range of lost steps: low values down to 1e-9 still count."""
    x, dy, a, ids = _problem(torch.float16, 128, 256, 128, 16, 2, seed=3)
    tiny = (dy.float() * 1e-5).half()  # about 1e-6: fp16 subnormals
    _check(x, tiny, a, ids, None, torch.zeros(128, 256, device=DEV), grad_dtype=torch.float32)
    big = (x.float() * 3000).half()    # low reaches past fp16's largest value
    _check(big, dy, a, ids, None, None, out_dtype=torch.float32, grad_dtype=torch.float32)


def test_many_adapters_and_long_order():
    t, g = 5000, 1500
    x, dy, a, ids = _problem(torch.bfloat16, t, 64, 64, 4, g, seed=4)
    plan = adapter_plan(ids.to(DEV).view(50, 100), g)
    y = adapter_linear(x, a, plan)
    s, ok = a.scale.double(), (ids >= 0) & (ids < g)
    i = ids.clamp(0, g - 1).to(DEV)
    low = torch.einsum("tk,trk->tr", x.double(), a.down.double()[i]) * s[i, None]
    ref = torch.einsum("tr,trn->tn", low, a.up.double()[i]) * ok.to(DEV)[:, None]
    mag = torch.einsum("tr,trn->tn", torch.einsum("tk,trk->tr", x.double().abs(), a.down.double().abs()[i])
                       * s[i, None], a.up.double().abs()[i])
    assert bool(((y.double() - ref).abs() <= _round_tol(ref, mag * (72 * 2.0**-23 + 2.0**-17),
                                                        torch.bfloat16)).all())


def test_refusals_on_the_device():
    x, dy, a, ids = _problem(torch.bfloat16, 10, 64, 32, 8, 3, seed=5)
    plan = adapter_plan(ids.to(DEV), 3)
    with pytest.raises(ValueError, match="tokens"):
        adapter_linear(x[:5], a, plan)
    with pytest.raises(ValueError, match="adapters"):
        adapter_linear(x, LowRankAdapters(down=a.down[:2], up=a.up[:2]), plan)
    with pytest.raises(TypeError):
        adapter_linear(x.half(), a, plan)
    with pytest.raises(ValueError):
        adapter_linear(x[:, :32], a, plan)
    with pytest.raises(TypeError):
        adapter_linear(x, a, plan, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="base"):
        adapter_linear(x, a, plan, base=torch.zeros(10, 31, device=DEV))
    with pytest.raises(ValueError, match="out"):
        adapter_linear(x, a, plan, out=torch.zeros(32, 10, device=DEV, dtype=torch.bfloat16).t())
    with pytest.raises(ValueError, match="8 bits"):
        adapter_linear_backward(dy, quantize_activations(x), a, plan)
    with pytest.raises(ValueError, match="low"):
        adapter_linear_backward(dy, x, a, plan, low=torch.zeros(10, 7, device=DEV))
    with pytest.raises(TypeError):
        adapter_plan(torch.zeros(4, device=DEV), 3)


def test_out_must_not_share_memory():
    x, dy, a, ids = _problem(torch.bfloat16, 10, 64, 64, 8, 3, seed=5)
    plan = adapter_plan(ids.to(DEV), 3)
    with pytest.raises(ValueError, match="share memory"):
        adapter_linear(x, a, plan, out=x)
    wide = torch.zeros(11, 64, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="share memory"):
        adapter_linear(x, a, plan, base=wide[1:], out=wide[:10])  # base, shifted by a row
    adapter_linear(x, a, plan, base=wide[:10], out=wide[1:11].clone())
    with pytest.raises(TypeError):
        AdaptedSparseLinear(BlockSparseLinear(bsr_from_tiles(
            torch.zeros(1, 64, 64, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV),
            torch.zeros(1, dtype=torch.int32, device=DEV), (64, 64))), 2, 8)


def test_two_calls_at_once():
    """Two batches on two streams through the same adapters, started together."""
    x, dy, a, _ = _problem(torch.bfloat16, 300, 512, 384, 16, 4, seed=13)
    ids = [torch.randint(-1, 4, (300,), device=DEV) for _ in range(2)]
    xs = [x, x.flip(0).contiguous()]

    def step(k):
        plan = adapter_plan(ids[k], 4)
        y, low = adapter_linear(xs[k], a, plan, return_low=True)
        return (y, *adapter_linear_backward(dy, xs[k], a, plan, low=low))

    ref = [step(0), step(1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    out = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[k].append(step(k))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for k in range(2) for o in out[k] for p, q in zip(o, ref[k]))


def test_backward_parts_and_checkpoint():
    x, dy, a, ids = _problem(torch.bfloat16, 150, 320, 128, 16, 3, seed=6)
    plan = adapter_plan(ids.to(DEV), 3)
    _, low = adapter_linear(x, a, plan, return_low=True)
    dx, dd, du = adapter_linear_backward(dy, x, a, plan, low=low)
    only_dx = adapter_linear_backward(dy, x, a, plan, need_dw=False)
    only_dw = adapter_linear_backward(dy, x, a, plan, low=low, need_dx=False)
    assert torch.equal(only_dx[0], dx) and only_dx[1] is None and only_dx[2] is None
    assert only_dw[0] is None and torch.equal(only_dw[1], dd) and torch.equal(only_dw[2], du)
    q = quantize_activations(x)
    kx, kd, ku = adapter_linear_backward(dy, q, a, plan, low=low, grad_dtype=torch.float32)
    assert torch.equal(kx, dx)
    back = dequantize_activations(q)
    _, _, rdl, mdl = _forward(dy, a, ids, None, swap=True)
    ref, mag = _wgrad(rdl, mdl, back, a, ids)
    assert bool(((kd.double() - ref).abs() <= _round_tol(ref, mag * ((128 + 150 + 4) * 2.0**-23 + 2.0**-23),
                                                         torch.float32)).all())
    assert torch.equal(ku, adapter_linear_backward(dy, x, a, plan, low=low, grad_dtype=torch.float32)[2])


def _layer(m, k, seed, checkpoint=None):
    gen = torch.Generator().manual_seed(seed)
    nbr, nbc = m // 64, k // 64
    pos = torch.sort(torch.randperm(nbr * nbc, generator=gen)[: nbr * nbc // 2]).values
    tiles = (torch.randn(pos.numel(), 64, 64, generator=gen) * 0.05).bfloat16().to(DEV)
    w = bsr_from_tiles(tiles, (pos // nbc).int().to(DEV), (pos % nbc).int().to(DEV), (m, k))
    dense = torch.zeros(nbr, nbc, 64, 64, dtype=torch.float64, device=DEV)
    dense[(pos // nbc).to(DEV), (pos % nbc).to(DEV)] = tiles.double()
    return w, dense.permute(0, 2, 1, 3).reshape(m, k), pos


@pytest.mark.parametrize("t", [1, 3, 200])
def test_beside_the_sparse_projection(t):
    w, dense, _ = _layer(256, 384, seed=7)
    x, dy, a, ids = _problem(torch.bfloat16, t, 384, 256, 16, 3, seed=8)
    plan = adapter_plan(ids.to(DEV), 3)
    for odt in (torch.bfloat16, torch.float32):
        y = adapted_sparse_linear(x, w, a, plan, out_dtype=odt)
        base, bmag = x.double() @ dense.t(), x.double().abs() @ dense.abs().t()
        ref, _, _, _ = _forward(x, a, ids, base)
        _, mag, _, _ = _forward(x, a, ids, bmag)
        slack = mag * ((384 + 384 + 20) * 2.0**-23 + _rest(odt))
        assert bool(((y.double() - ref).abs() <= _round_tol(ref, slack, odt)).all())
    with pytest.raises(ValueError):
        adapted_sparse_linear(x, w, LowRankAdapters(down=a.up, up=a.down), plan)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_model_step(checkpoint):
    """ids -> scaled lookup -> sparse layer with adapters (input kept in 8 bits) -> gradients of all four parameters."""
    t, m, k = 96, 256, 384
    w, dense, pos = _layer(m, k, seed=9)
    torch.manual_seed(0)
    emb = ScaledEmbedding(50, k, scale=2.0, dtype=torch.bfloat16, device=DEV)
    layer = AdaptedSparseLinear(BlockSparseLinear(w, checkpoint=checkpoint), 3, 8, scale=torch.tensor([1.0, 0.5, 2.0]))
    x0 = emb(torch.arange(5, device=DEV))
    plan0 = adapter_plan(torch.arange(5, device=DEV) % 3, 3)
    assert torch.equal(layer(x0, plan0), layer.layer(x0))  # a new adapter changes nothing
    with torch.no_grad():
        layer.up.normal_(std=0.3)
    ids = torch.randint(0, 50, (t,), device=DEV)
    req = torch.randint(-1, 3, (t,), device=DEV)
    plan = adapter_plan(req, 3)
    dy = (torch.randn(t, m, device=DEV) * 0.1).bfloat16()
    x = emb(ids)
    y = layer(x, plan)
    y.backward(dy)
    xd = x.detach()
    a = layer.adapters()
    base = xd.double() @ dense.t()
    ref, _, rl, ml = _forward(xd, a, req, base)
    _, mag, _, _ = _forward(xd, a, req, xd.double().abs() @ dense.abs().t())
    assert bool(((y.double() - ref).abs() <= _round_tol(ref, mag * (800 * 2.0**-23 + 2.0**-17),
                                                        torch.bfloat16)).all())
    kept = dequantize_activations(quantize_activations(xd)) if checkpoint else xd
    rx, _, rdl, mdl = _forward(dy, a, req, dy.double() @ dense, swap=True)
    _, mx, _, _ = _forward(dy, a, req, dy.double().abs() @ dense.abs(), swap=True)
    dref, dmag = _wgrad(rdl, mdl, kept, a, req)
    uref, umag = _wgrad(rl, ml, dy, a, req)
    half = 2.0**-8
    for got, ref, mag, terms in ((layer.down.grad, dref, dmag, m + t), (layer.up.grad, uref, umag, k + t)):
        assert bool(((got.double() - ref).abs() <= _round_tol(ref, mag * (terms * 2.0**-23 + 2.0**-17),
                                                              torch.bfloat16)).all())
    full = (dy.double().t() @ kept.double()).view(m // 64, 64, k // 64, 64).permute(0, 2, 1, 3).reshape(-1, 64, 64)
    fmag = (dy.double().abs().t() @ kept.double().abs()).view(m // 64, 64, k // 64, 64).permute(0, 2, 1, 3).reshape(
        -1, 64, 64)
    bref, bmag = full[pos.to(DEV)], fmag[pos.to(DEV)]
    assert bool(((layer.layer.blocks.grad.double() - bref).abs() <= _round_tol(bref, bmag * t * 2.0**-23,
                                                                               torch.bfloat16)).all())
    # the table's gradient sums dX (rounded to bf16) over tokens and rounds once more
    eref = torch.zeros(50, k, dtype=torch.float64, device=DEV).index_add_(0, ids, rx * 2)
    slack = torch.zeros_like(eref).index_add_(0, ids, 2 * _round_tol(rx, mx * (700 * 2.0**-23 + 2.0**-17),
                                                                     torch.bfloat16) + rx.abs() * t * 2.0**-23)
    assert bool(((emb.weight.grad.double() - eref).abs() <= slack + (eref.abs() + slack) * half * 1.01).all())


def test_gradient_against_differences():
    """The loss is linear in up and, with up fixed, in down: a difference of any size gives the derivative."""
    x, dy, a, ids = _problem(torch.bfloat16, 60, 64, 64, 8, 2, seed=10)
    plan = adapter_plan(ids.to(DEV), 2)
    _, low = adapter_linear(x, a, plan, return_low=True)
    _, dd, du = adapter_linear_backward(dy, x, a, plan, low=low, grad_dtype=torch.float32)

    def loss(down, up):
        y = adapter_linear(x, LowRankAdapters(down=down, up=up, scale=a.scale), plan, out_dtype=torch.float32)
        return (y.double() * dy.double()).sum().item()

    at = loss(a.down, a.up)
    for name, grad in (("down", dd), ("up", du)):
        flat = grad.flatten()
        i = int(flat.abs().argmax())
        p = {"down": a.down.clone(), "up": a.up.clone()}
        old = p[name].flatten()[i].item()
        p[name].view(-1)[i] = old + 1.0
        h = p[name].flatten()[i].item() - old  # the step that bf16 took
        diff = (loss(p["down"], p["up"]) - at) / h
        assert abs(diff - flat[i].item()) <= 1e-3 * abs(flat[i].item())  # 64 + 60 terms of 2^-23, and 3 roundings


def test_streams_and_graphs():
    x, dy, a, ids = _problem(torch.bfloat16, 70, 256, 192, 16, 4, seed=11)
    ids = ids.to(DEV)
    base = torch.randn(70, 192, device=DEV).bfloat16()

    def step():
        plan = adapter_plan(ids, 4)
        y, low = adapter_linear(x, a, plan, base=base, return_low=True)
        return (y, *adapter_linear_backward(dy, x, a, plan, low=low))

    ref = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(ref, got))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
        graphs.append((g, out))
    x.normal_()
    ids.copy_(torch.randint(-1, 4, (70,), device=DEV))
    ref = step()
    for _, out in graphs:
        for t in out:
            t.fill_(float("nan"))
    for _ in range(2):
        for g, _out in graphs:
            g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(p, q) for p, q in zip(ref, out))


def test_captured_training_step_beside_an_eager_one():
    """A captured forward and backward of the module while an eager graph of the same parameters is alive."""
    w, _, _ = _layer(128, 192, seed=12)
    layer = AdaptedSparseLinear(BlockSparseLinear(w, checkpoint="int8"), 2, 8)
    with torch.no_grad():
        layer.up.normal_(std=0.3)
    x = torch.randn(40, 192, device=DEV).bfloat16()
    dy = torch.randn(40, 128, device=DEV).bfloat16()
    plan = adapter_plan(torch.arange(40, device=DEV) % 3 - 1, 2)
    params = [layer.layer.blocks, layer.down, layer.up]

    def step():
        xi = x.detach().requires_grad_()
        return torch.autograd.grad(layer(xi, plan), [xi, *params], dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = step()
    alive = layer(x, plan)  # an eager graph of the same leaves
    x.normal_()
    ref = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ref, out))
    del alive


def test_offsets_pass_32_bits():
    """More than 2^31 values of X and of dX: the last tokens are read and written where they belong."""
    t, k = 66_000, 32_768
    x = torch.zeros(t, k, dtype=torch.bfloat16, device=DEV)
    x[-1], x[-2, 5] = 1.0, 2.0
    down = torch.full((2, 4, k), 2.0**-10, dtype=torch.bfloat16, device=DEV)
    up = torch.ones(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    a = LowRankAdapters(down=down, up=up)
    ids = torch.full((t,), -1, device=DEV)
    ids[-1], ids[-2], ids[3] = 1, 0, 0
    plan = adapter_plan(ids, 2)
    y, low = adapter_linear(x, a, plan, return_low=True)  # low of the last: 32768 * 2^-10 = 32
    assert low[-1].tolist() == [32.0] * 4 and low[-2].tolist() == [2.0**-9] * 4
    assert y[-1].unique().tolist() == [128.0] and bool((y[:-2] == 0).all())
    dy = torch.ones(t, 64, dtype=torch.bfloat16, device=DEV)
    dx, dd, du = adapter_linear_backward(dy, x, a, plan, low=low)
    # dlow = 64 for the three tokens with an adapter, dX = 4 * 64 * 2^-10
    assert dx[-1].unique().tolist() == [0.25] and dx[3].unique().tolist() == [0.25] and int(dx[4].count_nonzero()) == 0
    assert dd[1].unique().tolist() == [64.0] and dd[0, 0, 5].item() == 128.0 and du[1].unique().tolist() == [32.0]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("gdt", [None, torch.float32])
def test_gradients_at_any_address(dt, gdt):
    """The library's entries write gradients that start beside a 16-byte boundary, and nothing around them."""
    t, k, n, r, g = 70, 64, 72, 6, 3
    gdt = gdt or dt
    x, dy, a, ids = _problem(dt, t, k, n, r, g, seed=9)
    plan = adapter_plan(ids.to(DEV), g)
    _, low = adapter_linear(x, a, plan, return_low=True)
    _, dd, du = adapter_linear_backward(dy, x, a, plan, low=low, grad_dtype=gdt)
    _, dlow = adapter_linear(dy, LowRankAdapters(down=a.up, up=a.down, scale=a.scale), plan, return_low=True)
    lib, code, gcode = _lib.lib(), _lib.kairo_dtype(dt), _lib.kairo_dtype(gdt)
    s = torch.cuda.current_stream().cuda_stream
    for off in (1, 3):
        both = [torch.full((want.numel() + 8,), 7.0, dtype=gdt, device=DEV) for want in (dd, du)]
        at = [b[off:].data_ptr() for b in both]
        _lib.check(lib.kairo_low_rank_wgrads(dlow.data_ptr(), low.data_ptr(), r, x.data_ptr(), k, k, dy.data_ptr(), n, n,
                                             code, plan.memory.data_ptr(), t, g, at[0], at[1], gcode, s), "wgrads")
        one = torch.full((dd.numel() + 8,), 7.0, dtype=gdt, device=DEV)
        _lib.check(lib.kairo_low_rank_wgrad(dlow.data_ptr(), r, x.data_ptr(), k, k, code, plan.memory.data_ptr(), t, g,
                                            one[off:].data_ptr(), gcode, s), "wgrad")
        for buf, want in ((both[0], dd), (both[1], du), (one, dd)):
            assert torch.equal(buf[off : off + want.numel()].view_as(want), want)
            assert bool((buf[:off] == 7).all()) and bool((buf[off + want.numel():] == 7).all())


@pytest.mark.parametrize("t", [32768, 32769])
@pytest.mark.parametrize("r", [16, 40])
def test_gradients_of_long_batches(t, r):
    """Sums of one sign, where truncation adds up, on both sides of the length up to which the units add up all tokens."""
    k, n = 72, 64
    gen = torch.Generator().manual_seed(r)
    x = (torch.rand(t, k, generator=gen) + 0.5).bfloat16().to(DEV)
    dy = (torch.rand(t, n, generator=gen) + 0.5).bfloat16().to(DEV)
    low = (torch.rand(t, r, generator=gen) + 0.5).to(DEV)
    a = LowRankAdapters(down=torch.zeros(1, r, k, dtype=torch.bfloat16, device=DEV),
                        up=torch.ones(1, r, n, dtype=torch.bfloat16, device=DEV))
    plan = adapter_plan(torch.zeros(t, dtype=torch.int32, device=DEV), 1)
    _, dd, du = adapter_linear_backward(dy, x, a, plan, low=low)
    dlow = dy.double().sum(1, keepdim=True).expand(t, r)
    # per 16 tokens and term at most one truncation inside the units and one of the sum
    lost = 2 * (t / 16) * 2 * 2.0**-23 if t <= 32768 else (t / 64 + 32) * 2.0**-23
    for got, ref, own in ((dd[0], dlow.t() @ x.double(), (n + 2) * 2.0**-23), (du[0], low.double().t() @ dy.double(), 0.0)):
        slack = ref * (lost + own + 2.0**-17)
        assert bool(((got.double() - ref).abs() <= _round_tol(ref, slack, torch.bfloat16)).all())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", [
    (3, 1, 1, 1, 1), (70, 2, 3, 2, 2), (64, 64, 65, 16, 1), (130, 1471, 334, 12, 4), (50, 333, 1025, 33, 2),
    (20, 131, 99, 128, 2), (300, 97, 129, 64, 3),
])
def test_odd_features(dt, case):
    """Rows that begin at any address; calls on NaN before each leave nothing behind that reaches a result."""
    t, k, n, r, g = case
    x, dy, a, ids = _problem(dt, t, k, n, r, g, seed=t + k)
    nan = LowRankAdapters(down=torch.full_like(a.down, float("nan")), up=torch.full_like(a.up, float("nan")))
    gen = torch.Generator().manual_seed(k)
    for base_t, out_t in ((None, None), (dt, torch.float32), (torch.float32, None)):
        base = base_dx = None
        if base_t is not None:
            wide = torch.randn(t, n + k + 3, generator=gen).to(base_t).to(DEV)
            base, base_dx = wide[:, 1 : n + 1], wide[:, n + 2 : n + 2 + k]
        plan = adapter_plan(torch.zeros(t, dtype=torch.int64, device=DEV), g)
        y = adapter_linear(torch.full_like(x, float("nan")), nan, plan)
        adapter_linear_backward(y, torch.full_like(x, float("nan")), nan, plan)
        _check(x, dy, a, ids, base, base_dx, out_dtype=out_t, grad_dtype=out_t)
