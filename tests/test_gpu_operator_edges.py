"""Corners of the operators around the linear layer on the device.

Plain implementations are in 64 bits.  Tolerances count half steps of the
output's type (torch.finfo(t).eps / 2 of the value) and, for a sum of n products in
fp32, n * 2^-23 of the sum of magnitudes.
"""

from __future__ import annotations

import pytest
import torch

from kairo_b200.ops import (
    AdaptedSparseLinear,
    BlockSparseLinear,
    LowRankAdapters,
    TokenOrder,
    adapter_linear,
    adapter_linear_backward,
    adapter_plan,
    bsr_from_tiles,
    dequantize_activations,
    embedding_grad,
    embedding_lookup,
    quantize_activations,
    sort_tokens,
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


def _adapted(m=256, k=320, checkpoint=None, seed=1, dt=torch.bfloat16):
    w, rows, cols = _weight(dt, m, k, seed=seed)
    torch.manual_seed(seed)
    layer = AdaptedSparseLinear(BlockSparseLinear(w, checkpoint=checkpoint), 3, 8, scale=torch.tensor([1.0, 0.5, 2.0]))
    with torch.no_grad():
        layer.up.normal_(std=0.3)
    x = torch.randn(70, k, device=DEV).to(dt)
    dy = (torch.randn(70, m, device=DEV) * 0.1).to(dt)
    plan = adapter_plan(torch.arange(70, device=DEV) % 4 - 1, 3)
    return layer, x, dy, plan


def _gradients(layer, x, dy, plan):
    """(dX, d_blocks, d_down, d_up) of one step; None where nothing asks for one."""
    for p in layer.parameters():
        p.grad = None
    xi = x.clone().requires_grad_()
    layer(xi, plan).backward(dy)
    return xi.grad, layer.layer.blocks.grad, layer.down.grad, layer.up.grad


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_frozen_parameters_of_an_adapted_layer(checkpoint):
    """Every subset of the parameters frozen, all of them too: what is left has the gradients of the whole."""
    layer, x, dy, plan = _adapted(checkpoint=checkpoint)
    params = [layer.layer.blocks, layer.down, layer.up]
    whole = _gradients(layer, x, dy, plan)
    for keep in range(8):
        for i, p in enumerate(params):
            p.requires_grad_(bool(keep >> i & 1))
        got = _gradients(layer, x, dy, plan)
        assert torch.equal(got[0], whole[0])
        for i in range(3):
            assert torch.equal(got[1 + i], whole[1 + i]) if keep >> i & 1 else got[1 + i] is None
    a = layer.adapters()
    dx, dd, du = adapter_linear_backward(dy, None, a, plan, need_dw=False)
    assert torch.equal(dx, adapter_linear_backward(dy, x, a, plan)[0]) and dd is None and du is None


def test_scale_of_the_forward_pass():
    """The gradients are those of the scale that the forward pass used, or autograd says that it was written."""
    layer, x, dy, plan = _adapted()
    ref = _gradients(layer, x, dy, plan)
    for p in layer.parameters():
        p.grad = None
    xi = x.clone().requires_grad_()
    y = layer(xi, plan)
    used = layer.scale
    layer.scale = torch.zeros_like(used)  # a reference pass without the adapters
    assert torch.equal(layer(x, plan), layer.layer(x))
    y.backward(dy)
    layer.scale = used
    got = xi.grad, layer.layer.blocks.grad, layer.down.grad, layer.up.grad
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    y = layer(xi, plan)
    layer.scale.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


@pytest.mark.parametrize("k", [320, 200, 72])
@pytest.mark.parametrize("pin", [False, True])
@pytest.mark.parametrize("tokens", [70, 1])
def test_checkpoint_under_offloading_hooks(k, pin, tokens):
    """What is kept survives a copy to the host and back, at widths that are no multiple of 16, too."""
    layer, x, dy, _ = _adapted(k=k, checkpoint="int8")
    x, dy = x[:tokens], dy[:tokens]
    plan = adapter_plan(torch.arange(tokens, device=DEV) % 4, 3)
    inner = layer.layer

    def plain():
        inner.blocks.grad = None
        inner(x).backward(dy)
        return inner.blocks.grad

    ref, ref_plain = _gradients(layer, x, dy, plan), plain()
    with torch.autograd.graph.save_on_cpu(pin_memory=pin):
        got, got_plain = _gradients(layer, x, dy, plan), plain()
    assert all(torch.equal(a, b) for a, b in zip(got, ref)) and torch.equal(got_plain, ref_plain)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone()):
        got, got_plain = _gradients(layer, x, dy, plan), plain()
    assert all(torch.equal(a, b) for a, b in zip(got, ref)) and torch.equal(got_plain, ref_plain)


def test_gradient_over_its_own_order_is_refused():
    ids = torch.arange(16, device=DEV) % 5
    order = sort_tokens(ids, 5)
    out = torch.zeros(5, 32, device=DEV)
    inside = out.view(-1)[:16].view(torch.int32)
    g = torch.ones(16, 32, device=DEV)
    for part in ("sorted_ids", "perm"):
        parts = {"sorted_ids": order.sorted_ids, "perm": order.perm}
        parts[part] = inside.copy_(parts[part])
        with pytest.raises(ValueError, match="share memory"):
            embedding_grad(g, TokenOrder(**parts, num_embeddings=5), 5, out=out)


@pytest.mark.parametrize("dt,d", [(torch.bfloat16, 2048), (torch.float32, 1024)])
@pytest.mark.parametrize("tokens", [4097, 5000, 40000])
def test_gradient_of_a_large_table(dt, d, tokens):
    """Only the last rows are zeroed beside the sort (some 48 to 116 MB of them): rows with and without tokens on
    both sides of the border, in a buffer that held NaN."""
    n = 40000  # 160 MB
    g = torch.Generator(device=DEV).manual_seed(tokens)
    grad = torch.randn(tokens, d, generator=g, device=DEV).to(dt)
    ids = torch.randint(-100, n + 100, (tokens,), generator=g, device=DEV)
    ids[:40], ids[-40:] = n - 1, 0
    out = torch.full((n, d), float("nan"), dtype=dt, device=DEV)
    assert embedding_grad(grad, ids, n, scale=0.5, out=out) is out
    ok = (ids >= 0) & (ids < n)
    used, row = torch.unique(ids[ok], return_inverse=True)
    ref = torch.zeros(used.numel(), d, dtype=torch.float64, device=DEV).index_add_(0, row, grad[ok].double() * 0.5)
    mag = torch.zeros_like(ref).index_add_(0, row, grad[ok].double().abs() * 0.5)
    # a sum of c fp32 values is off by at most (c - 1) * 2^-24 of the magnitudes; then the scale's product
    tol = mag * (torch.bincount(row)[:, None] + 3) * 2.0**-24
    assert bool(((out[used].double() - ref).abs() <= tol + (ref.abs() + tol) * _half(dt) * 1.01 + 1e-30).all())
    rest = torch.ones(n, dtype=torch.bool, device=DEV)
    rest[used] = False
    assert int(rest.sum()) > 0 and bool((out[rest] == 0).all())


@pytest.mark.parametrize("wt,ot", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
                                   (torch.float16, torch.float32)])
@pytest.mark.parametrize("d", [64, 1000, 2048, 37])
@pytest.mark.parametrize("tokens", [19999, 20480, 40001])
def test_lookup_of_long_lists(wt, ot, d, tokens):
    """Four rows of a thread under way: every width, ids outside the table, a last group that is not whole."""
    n = 700
    g = torch.Generator(device=DEV).manual_seed(d)
    w = torch.randn(n, d, generator=g, device=DEV).to(wt)
    ids = torch.randint(-3, n + 3, (tokens,), generator=g, device=DEV)
    buf = torch.full((tokens + 1, d), 7.0, dtype=ot, device=DEV)
    embedding_lookup(w, ids, scale=1.7, out=buf[:tokens])
    ok = (ids >= 0) & (ids < n)
    ref = w.double()[ids.clamp(0, n - 1)] * 1.7 * ok[:, None]
    # half a step of the output, of the fp32 product and of 1.7 in fp32
    tol = ref.abs() * (_half(ot) * 1.001 + 2 * 2.0**-24) + torch.finfo(ot).smallest_normal * _half(ot) * 2
    assert bool(((buf[:tokens].double() - ref).abs() <= tol).all()) and bool((buf[tokens] == 7).all())


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k,n", [(4096, 4096), (4104, 3592), (8192, 64), (72, 8192), (4097, 3601)])
@pytest.mark.parametrize("tokens,rank", [(1, 16), (20, 16), (20, 40), (3, 128)])
def test_wide_layers_of_few_tokens(dt, k, n, tokens, rank):
    """Eight CTAs to a tile: features in 64 x 8 x 8 parts, whole and not, forward and backward against 64 bits."""
    gen = torch.Generator(device=DEV).manual_seed(k + n + tokens)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    x, dy = rand(tokens, k).to(dt), (rand(tokens, n) * 0.1).to(dt)
    down, up = (rand(3, rank, k) * k**-0.5).to(dt), (rand(3, rank, n) * rank**-0.5).to(dt)
    scale = torch.tensor([1.0, 0.5, 2.0], device=DEV)
    ids = torch.arange(tokens, device=DEV) % 4 - int(tokens > 1)  # -1: none
    base, base_dx = rand(tokens, n).to(dt), rand(tokens, k).to(dt)
    a, plan = LowRankAdapters(down=down, up=up, scale=scale), adapter_plan(ids, 3)
    y, low = adapter_linear(x, a, plan, base=base, return_low=True)
    dx, dd, du = adapter_linear_backward(dy, x, a, plan, low=low, base_dx=base_dx, grad_dtype=torch.float32)

    mine = ((ids >= 0) & (ids < 3)).double() * scale.double()[ids.clamp(0, 2)]
    at = ids.clamp(0, 2)

    def forward(v, first, second, start, f=lambda t: t):
        v, first, second = f(v.double()), f(first.double())[at], f(second.double())[at]
        lo = torch.einsum("tk,trk->tr", v, first) * mine[:, None]
        return lo, f(start.double()) + torch.einsum("tr,trn->tn", lo, second)

    def inside(got, ref, mag, terms, rest, t):
        slack = mag * (terms * 2.0**-23 + rest)
        tiny = torch.finfo(t).smallest_normal * _half(t) * 2
        assert bool(((got.double() - ref).abs() <= slack + (ref.abs() + slack) * _half(t) * 1.01 + tiny).all())

    rl, ry = forward(x, down, up, base)
    ml, my = forward(x, down, up, base, torch.abs)
    rdl, rx = forward(dy, up, down, base_dx)
    mdl, mx = forward(dy, up, down, base_dx, torch.abs)
    inside(low, rl, ml, k + 2, 0.0, torch.float32)
    inside(y, ry, my, k + rank + 4, 2.0**-17, dt)
    inside(dx, rx, mx, n + rank + 4, 2.0**-17, dt)
    one = torch.nn.functional.one_hot(at, 3).double() * ((ids >= 0) & (ids < 3))[:, None]
    for got, s, sm, z, terms in ((dd, rdl, mdl, x, n), (du, rl, ml, dy, k)):
        ref = torch.einsum("tg,tr,tk->grk", one, s, z.double())
        mag = torch.einsum("tg,tr,tk->grk", one, sm, z.double().abs())
        inside(got, ref, mag, terms + tokens + 4, 2.0**-23, torch.float32)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_layers_without_gradients(checkpoint):
    """The same bits with and without a graph; without one nothing is allocated for a backward pass."""
    layer, x, dy, plan = _adapted(checkpoint=checkpoint)
    want, inner = layer(x, plan), layer.layer(x)
    with torch.no_grad():
        assert torch.equal(layer(x, plan), want) and torch.equal(layer.layer(x), inner)


@pytest.mark.parametrize("ot", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 31, 40, 256])
@pytest.mark.parametrize("n,d", [(70, 40), (100_000, 36), (3000, 517)])
def test_short_lists_accumulate(ot, tokens, n, d):
    """A short list added to a caller's rows: base + sum with one rounding, other rows keep their bits, and the
    same bits as through the sorted order."""
    g = torch.Generator(device=DEV).manual_seed(tokens + n)
    grad = torch.randn(tokens, d, generator=g, device=DEV)
    ids = torch.randint(-2, n + 2, (tokens,), generator=g, device=DEV)
    ids[: tokens // 3] = 5  # one id in several parts
    ok = (ids >= 0) & (ids < n)
    used = torch.zeros(n, dtype=torch.bool, device=DEV)
    used[ids[ok]] = True
    base = torch.randn(n, d, generator=g, device=DEV).to(ot)
    base[~used] = float("nan")
    wide = torch.full((n, d + 5), 3.0, dtype=ot, device=DEV)
    out = wide[:, :d]
    out.copy_(base)
    assert embedding_grad(grad, ids, n, scale=0.25, out=out, accumulate=True) is out
    other = base.clone()
    embedding_grad(grad, sort_tokens(ids, n), n, scale=0.25, out=other, accumulate=True)
    assert torch.equal(out[used], other[used]) and bool(other[~used].isnan().all())
    assert bool(out[~used].isnan().all()) and bool((wide[:, d:] == 3).all())
    ref = torch.zeros(n, d, dtype=torch.float64, device=DEV).index_add_(0, ids[ok], grad[ok].double() * 0.25)
    mag = torch.zeros(n, d, dtype=torch.float64, device=DEV).index_add_(0, ids[ok], grad[ok].double().abs() * 0.25)
    count = torch.zeros(n, dtype=torch.float64, device=DEV).index_add_(0, ids[ok], torch.ones(
        int(ok.sum()), dtype=torch.float64, device=DEV))
    ref, mag = ref[used] + base[used].double(), mag[used] + base[used].double().abs()
    # a sum of count fp32 values, the scale's product and the sum with the base
    s = mag * (count[used][:, None] + 3) * 2.0**-24
    assert bool(((out[used].double() - ref).abs() <= s + (ref.abs() + s) * _half(ot) * 1.01 + 1e-38).all())


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k,n", [(128, 64), (131, 67)])
def test_infinities_in_the_factors(dt, k, n):
    """An infinity makes what it enters non-finite and changes nothing else, forward and backward."""
    gen = torch.Generator(device=DEV).manual_seed(k)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(dt)  # noqa: E731
    x, dy, down, up = rand(48, k), rand(48, n), rand(3, 8, k), rand(3, 8, n)
    ids = torch.arange(48, device=DEV) % 4 - 1
    plan = adapter_plan(ids, 3)

    def step(x, dy, down, up):
        a = LowRankAdapters(down=down, up=up)
        y, low = adapter_linear(x, a, plan, return_low=True)
        return (y, *adapter_linear_backward(dy, x, a, plan, low=low))

    clean = step(x, dy, down, up)
    inf = float("inf")
    u = up.clone()
    u[1, 2, 9] = inf  # enters column 9 of y, dlow and so dX and d_down of adapter 1's tokens
    y, dx, dd, du = step(x, dy, down, u)
    mine = ids == 1
    col = torch.zeros(n, dtype=torch.bool, device=DEV)
    col[9] = True
    assert not bool(y[mine][:, col].isfinite().any()) and torch.equal(y[:, ~col], clean[0][:, ~col])
    assert torch.equal(y[~mine], clean[0][~mine]) and torch.equal(dx[~mine], clean[1][~mine])
    assert not bool(dx[mine].isfinite().any()) and torch.equal(du, clean[3])
    assert not bool(dd[1, 2].isfinite().any()) and torch.equal(dd[[0, 2]], clean[2][[0, 2]])
    z = x.clone()
    z[6, 5] = -inf  # a token of adapter 1: its y and d_up, and one column of d_down
    y, dx, dd, du = step(z, dy, down, up)
    rest = torch.arange(48, device=DEV) != 6
    assert not bool(y[6].isfinite().any()) and torch.equal(y[rest], clean[0][rest]) and torch.equal(dx, clean[1])
    assert not bool(dd[1][:, 5].isfinite().any()) and not bool(du[1].isfinite().any())
    assert torch.equal(dd[[0, 2]], clean[2][[0, 2]]) and torch.equal(du[[0, 2]], clean[3][[0, 2]])
    keep = torch.arange(k, device=DEV) != 5
    assert torch.equal(dd[1][:, keep], clean[2][1][:, keep])


@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("k", [320, 200])
def test_an_empty_batch_through_the_layer(checkpoint, k):
    layer, x, dy, _ = _adapted(k=k, checkpoint=checkpoint)
    plan = adapter_plan(torch.zeros(0, dtype=torch.int64, device=DEV), 3)
    dx, db, dd, du = _gradients(layer, x[:0], dy[:0], plan)
    assert dx.shape == (0, k)
    assert bool((db == 0).all()) and bool((dd == 0).all()) and bool((du == 0).all())


def test_results_beside_their_inputs():
    """Columns of one wider matrix: the input on the left, base and result in place on the right."""
    layer, x, dy, plan = _adapted()
    a = layer.adapters()
    base = torch.randn(70, 256, device=DEV).bfloat16()
    wide = torch.cat([x, base, torch.zeros_like(base)], dim=1)
    xv, bv, ov = wide[:, :320], wide[:, 320:576], wide[:, 576:]
    want = adapter_linear(x, a, plan, base=base)
    assert torch.equal(adapter_linear(xv, a, plan, base=bv, out=ov), want)
    assert torch.equal(wide[:, :320], x) and torch.equal(bv, base)
    assert torch.equal(adapter_linear(xv, a, plan, base=bv, out=bv), want) and torch.equal(wide[:, :320], x)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", [131080, 131073, 1 << 19, (1 << 19) + 8, 1 << 20])
@pytest.mark.parametrize("t,rank", [(2, 20), (2100, 8)])
def test_long_contractions_to_16_bits(dt, k, t, rank):
    """16-bit results without low stay at their own rounding, on both sides of the length of one sum."""
    if t > 100 and k > 140_000:
        t = 60
    gen = torch.Generator(device=DEV).manual_seed(k + rank)
    x = (torch.rand(t, k, generator=gen, device=DEV) + 0.5).to(dt)
    down = ((torch.rand(2, rank, k, generator=gen, device=DEV) + 0.5) * 2**-14).to(dt)
    up = torch.full((2, rank, 72), 2.0**-6, dtype=dt, device=DEV)
    ids = torch.arange(t, device=DEV) % 2
    y = adapter_linear(x, LowRankAdapters(down=down, up=up), adapter_plan(ids, 2))
    low = torch.zeros(t, rank, dtype=torch.float64, device=DEV)
    for g in range(2):
        for c in range(0, k, 1 << 17):
            low[ids == g] += x[ids == g, c : c + (1 << 17)].double() @ down[g, :, c : c + (1 << 17)].double().t()
    want = low.sum(1, keepdim=True).expand(t, 72) * 2.0**-6
    # 128 products in a part, two truncations each; low in two terms; sums over parts, warps, CTAs and ranks
    slack = want * (128 * 2 * 2.0**-23 + 2.0**-17 + (rank + 24) * 2.0**-23)
    assert bool(((y.double() - want).abs() <= slack + (want + slack) * _half(dt) * 1.01).all())
