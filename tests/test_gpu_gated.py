"""Gated block-sparse projection and its gradients, against the formulas in 64 bits.

Bounds.  A sum of n products with absolute terms A, added 16 at a time, is off
by at most n / 16 * 2^-22 * A (each step truncates).  act is off by 2^-20 of its
arguments' size, its slope by 2^-19.  H, dG and dU are rounded to 16 bits once (h
= eps / 2), and the results again.
"""

from __future__ import annotations

import math

import pytest
import torch

from kairo_b200 import _lib, ops
from kairo_b200.ops import bsr_from_tiles

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
ACTS = ["silu", "gelu", "gelu_tanh", "relu"]


def act64(g, act):
    g = g.detach().requires_grad_(True)
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
         "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[act](g)
    (d,) = torch.autograd.grad(f.sum(), g)
    return f.detach(), d


def weight(m, k, b, keep, dtype, g, shuffle=False, pos=None):
    nbr, nbc = -(-m // b), -(-k // b)
    if pos is None:
        pos = torch.nonzero(torch.rand(nbr * nbc, generator=g, device="cuda") < keep)[:, 0]
    if shuffle:
        pos = pos[torch.randperm(pos.numel(), generator=g, device="cuda")]
    blocks = (torch.randn(pos.numel(), b, b, generator=g, device="cuda") * (max(keep, 0.05) * k) ** -0.5).to(dtype)
    a = bsr_from_tiles(blocks, (pos // nbc).int(), (pos % nbc).int(), (m, k))
    dense = torch.zeros(nbr, nbc, b, b, dtype=torch.float64, device="cuda")
    dense[pos // nbc, pos % nbc] = blocks.double()
    return a, dense.transpose(1, 2).reshape(nbr * b, nbc * b)[:m, :k], pos


def blocks_of(dense, a):
    """The blocks of ``a``'s pattern, in BSR order, of a dense matrix."""
    m, k = dense.shape
    b = a.block_size[0]
    full = torch.nn.functional.pad(dense, (0, -k % b, 0, -m % b))
    rows = torch.repeat_interleave(torch.arange(a.nbr, device="cuda"), (a.row_ptr[1:] - a.row_ptr[:-1]).long())
    return full.view(full.shape[0] // b, b, -1, b)[rows, :, a.col_idx.long(), :]


def within(name, got, want, tol):
    assert torch.isfinite(got.double()).all(), f"{name} is not finite"
    off = (got.double() - want).abs() - tol
    worst = off.max() if off.numel() else torch.tensor(-1.0)
    assert worst <= 0, f"{name}: {worst.item():.3g} over its bound"


def check(x, dh, wg, wu, gate, up, act, h, dx, dgate, dup, skip_h=False):
    eps = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2
    xd, dhd = x.double(), dh.double()
    step = (x.shape[1] / 16 + 1) * 2.0**-22
    g, u = xd @ wg.t(), xd @ wu.t()
    eg, eu = step * (xd.abs() @ wg.abs().t()), step * (xd.abs() @ wu.abs().t())
    f, d = act64(g, act)
    ef = 1.2 * eg + 2.0**-20 * g.abs()      # |act'| <= 1.13
    ed = 1.1 * eg + 2.0**-19 * (1 + g.abs())  # |act''| <= 1.1 where act is smooth
    if act == "relu":
        ed = torch.where(g.abs() <= eg, 1.0, 0.0)
    e = u.abs() * ef + f.abs() * eu + ef * eu
    if not skip_h:
        within("H", h, f * u, e * (1 + eps) + eps * (f * u).abs() + tiny)
    dg, du = dhd * u * d, dhd * f
    edg = dhd.abs() * (u.abs() * ed + d.abs() * eu + ed * eu)
    edu = dhd.abs() * ef
    edg = edg * (1 + eps) + eps * dg.abs() + tiny
    edu = edu * (1 + eps) + eps * du.abs() + tiny
    sm, sn = (wg.shape[0] / 8 + 1) * 2.0**-22, (x.shape[0] / 16 + 1) * 2.0**-22
    want = dg @ wg + du @ wu
    terms = dg.abs() @ wg.abs() + du.abs() @ wu.abs()
    within("dX", dx, want, (edg @ wg.abs() + edu @ wu.abs()) * (1 + sm) + sm * terms + eps * 1.01 * want.abs() + tiny)
    for name, got, p, q, a in (("d_gate", dgate, dg, edg, gate), ("d_up", dup, du, edu, up)):
        want = p.t() @ xd
        tol = (q.t() @ xd.abs()) * (1 + sn) + sn * (p.abs().t() @ xd.abs()) + eps * 1.01 * want.abs() + tiny
        within(name, got, blocks_of(want, a), blocks_of(tol, a))


def case(tokens, m, k, b, dtype, act="silu", keep=0.4, shared=False, seed=0, shuffle=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    gate, wg, pos = weight(m, k, b, keep, dtype, g, shuffle)
    up, wu, _ = weight(m, k, b, keep, dtype, g, shuffle, pos if shared else None)
    x = torch.randn(tokens, k, generator=g, device="cuda").to(dtype)
    dh = torch.randn(tokens, m, generator=g, device="cuda").to(dtype)
    return x, dh, gate, up, wg, wu


def run_case(*args, **kw):
    x, dh, gate, up, wg, wu = case(*args, **kw)
    act = kw.get("act", "silu")
    w = ops.gated_weights(gate, up)
    h = ops.sparse_gated_linear(x, w, activation=act, check=True)
    dx, db = ops.sparse_gated_linear_backward(dh, x, w, activation=act, check=True)
    assert h.dtype == dx.dtype == db.dtype == x.dtype and db.shape == w.blocks.shape
    check(x, dh, wg, wu, gate, up, act, h, dx, *w.split(db))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b", [64, 32, 16])
@pytest.mark.parametrize("tokens", [1, 2, 8, 9, 16, 17, 31, 32, 33, 128, 129, 255, 257, 511, 600])
def test_tokens(tokens, b, dtype):
    run_case(tokens, 192, 256, b, dtype)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("tokens,m,k,b,keep,shared", [(5, 520, 1000, 64, 0.5, False), (300, 520, 1000, 64, 0.5, True),
                                                      (70, 33, 777, 32, 0.3, False), (700, 100, 129, 16, 0.9, False),
                                                      (260, 640, 2048, 64, 0.05, False), (40, 1, 1, 16, 1.0, True)])
def test_shapes(tokens, m, k, b, keep, shared, act):
    run_case(tokens, m, k, b, torch.bfloat16 if tokens % 20 else torch.float16, act=act, keep=keep, shared=shared)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [9, 16, 17, 32, 33, 64, 65])
def test_many_rows(tokens, dtype):
    """256 block-rows and more: the blocks are streamed."""
    run_case(tokens, 64 * 259 - 7, 136, 64, dtype, act="silu")


@pytest.mark.parametrize("tokens", [20, 64, 65, 128, 129, 256])
@pytest.mark.parametrize("b", [64, 16])
def test_more_rows_than_places(tokens, b):
    """Several block-rows for each resident CTA, some of them empty."""
    run_case(tokens, b * 700 - 5, 2 * b + 8, b, torch.float16, act="gelu", keep=0.4)


@pytest.mark.parametrize("tokens,b,nbc", [(1, 64, 70), (3, 16, 300), (20, 32, 67), (40, 32, 67), (50, 16, 80),
                                          (600, 64, 70), (300, 16, 140)])
def test_long_rows(tokens, b, nbc):
    """Rows of more entries than a window holds."""
    run_case(tokens, 2 * b, b * nbc, b, torch.bfloat16, keep=0.95, act="gelu")


@pytest.mark.parametrize("tokens", [1, 12, 50, 300])
@pytest.mark.parametrize("b", [64, 32, 16])
def test_empty_parts(tokens, b):
    """Rows that keep nothing, a weight that keeps nothing, two that keep nothing."""
    m, k = 5 * b - 3, 4 * b
    g = torch.Generator(device="cuda").manual_seed(3)
    some = torch.tensor([0, 1, 3, 9, 10, 17], device="cuda")  # rows 0, 2 and 4 of 5
    none = some[:0]
    for pg, pu in ((some, some), (some, none), (none, some), (none, none), (some[:2], some[3:])):
        gate, wg, _ = weight(m, k, b, 0.5, torch.bfloat16, g, pos=pg)
        up, wu, _ = weight(m, k, b, 0.5, torch.bfloat16, g, pos=pu)
        w = ops.gated_weights(gate, up)
        x = torch.randn(tokens, k, generator=g, device="cuda").bfloat16()
        dh = torch.randn(tokens, m, generator=g, device="cuda").bfloat16()
        out = torch.full((tokens + 1, m), 7.0, device="cuda").bfloat16()
        h = ops.sparse_gated_linear(x, w, out=out[:tokens], check=True)
        assert (out[tokens] == 7).all()  # the row behind the last token is left as it was
        dx, db = ops.sparse_gated_linear_backward(dh, x, w, check=True)
        check(x, dh, wg, wu, gate, up, "silu", h, dx, *w.split(db))


@pytest.mark.parametrize("tokens", [5, 40, 300])
def test_layouts(tokens):
    """Blocks out of order, rows of a wider matrix, rows at odd addresses, a transposed X, a broadcast dH."""
    x, dh, gate, up, wg, wu = case(tokens, 200, 203, 32, torch.bfloat16, shuffle=True)
    w = ops.gated_weights(gate, up)
    assert gate.blk_idx is not None
    g, u = w.matrices()
    assert torch.equal(g.col_idx, gate.col_idx) and torch.equal(u.row_ptr, up.row_ptr)
    want = ops.sparse_gated_linear(x, w)
    wide = torch.full((tokens, 512), 9.0, device="cuda").bfloat16()
    for at in (0, 1, 8):
        wide[:, at:at + 203] = x
        assert torch.equal(ops.sparse_gated_linear(wide[:, at:at + 203], w, check=True), want)
    assert torch.equal(ops.sparse_gated_linear(x.t().contiguous().t(), w), want)
    for at in (0, 3):
        out = torch.full((tokens, 256), 5.0, device="cuda").bfloat16()
        ops.sparse_gated_linear(x, w, out=out[:, at:at + 200])
        assert torch.equal(out[:, at:at + 200], want) and (out[:, at + 200:] == 5).all() and (out[:, :at] == 5).all()
    row = torch.randn(1, 200, device="cuda").bfloat16().expand(tokens, 200)
    for d in (row, dh.t().contiguous().t()):
        a = ops.sparse_gated_linear_backward(d, x, w)
        b = ops.sparse_gated_linear_backward(d.contiguous(), x, w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    dx, db = ops.sparse_gated_linear_backward(dh, x, w, need_dw=False)
    assert db is None
    dx2, db = ops.sparse_gated_linear_backward(dh, x, w, need_dx=False)
    assert dx2 is None
    dx3, db32 = ops.sparse_gated_linear_backward(dh, x, w, dw_dtype=torch.float32)
    assert torch.equal(dx, dx3) and db32.dtype == torch.float32 and torch.equal(db32.bfloat16(), db)


def test_no_tokens():
    x, dh, gate, up, wg, wu = case(4, 100, 100, 32, torch.float16)
    w = ops.gated_weights(gate, up)
    assert ops.sparse_gated_linear(x[:0], w).shape == (0, 100)
    dx, db = ops.sparse_gated_linear_backward(dh[:0], x[:0], w)
    assert dx.shape == (0, 100) and db.shape == w.blocks.shape and not db.any()


@pytest.mark.parametrize("act", ["gelu_tanh", "relu"])
def test_huge_values(act):
    """Sums of the order of 1e20, whose squares are infinite: what is far from zero has a slope of 0 or 1."""
    x, dh, gate, up, wg, wu = case(20, 64, 64, 32, torch.bfloat16, act=act, keep=1.0)
    x = x * 2.0**66
    w = ops.gated_weights(gate, up)
    h = ops.sparse_gated_linear(x, w, activation=act)
    small = dh * 2.0**-100
    dx, db = ops.sparse_gated_linear_backward(small, x, w, activation=act)
    check(x, small, wg, wu, gate, up, act, h.where(torch.isfinite(h), 0), dx, *w.split(db), skip_h=True)
    g, u = x.double() @ wg.t(), x.double() @ wu.t()
    assert torch.equal(h == 0, (g < 0) | (u == 0)) or act == "gelu_tanh"
    # a NaN stays one
    x[3, 0] = float("nan")
    assert torch.isnan(ops.sparse_gated_linear(x, w, activation=act)[3]).all()


@pytest.mark.parametrize("tokens", [6, 40, 300])
@pytest.mark.parametrize("b", [64, 16])
def test_not_finite(tokens, b):
    """An infinity or a NaN reaches the rows that keep a block in its column, of its token, and no others."""
    x, dh, gate, up, wg, wu = case(tokens, 6 * b, 5 * b, b, torch.bfloat16, keep=0.3)
    w = ops.gated_weights(gate, up)
    want = ops.sparse_gated_linear(x, w)
    bad = x.clone()
    bad[2, 0], bad[4, 3 * b + 1] = float("nan"), float("inf")
    got = ops.sparse_gated_linear(bad, w)
    keeps = (wg.view(6, b, 5, b).abs().amax((1, 3)) + wu.view(6, b, 5, b).abs().amax((1, 3))) > 0  # row, column
    for token, col in ((2, 0), (4, 3)):
        hit = keeps[:, col].repeat_interleave(b)
        assert not torch.isfinite(got[token, hit]).any()
        assert torch.equal(got[token, ~hit], want[token, ~hit])
    others = [t for t in range(tokens) if t not in (2, 4)]
    assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("tokens", [4, 20, 50, 300])
@pytest.mark.parametrize("b", [64, 32])
def test_malformed_entries(tokens, b):
    """An entry out of range is recorded and read nowhere; the next call is clean."""
    x, dh, gate, up, wg, wu = case(tokens, 260 * b if tokens == 20 else 3 * b, 4 * b, b, torch.bfloat16, keep=0.9)
    w = ops.gated_weights(gate, up)
    want = ops.sparse_gated_linear(x, w, check=True)
    for field, value in ((0, 4), (0, -1), (1, w.blocks.shape[0]), (2, 1 << 30), (1, -2)):
        kept = w.entries[1].clone()
        w.entries[1, field] = value
        with pytest.raises(_lib.KairoDeviceError) as e:
            ops.sparse_gated_linear(x, w, check=True)
        assert e.value.code & 0xFF == _lib.DEVERR_BAD_INDEX
        ops.sparse_gated_linear(x, w)
        assert ops.pending_device_error() & 0xFF == _lib.DEVERR_BAD_INDEX
        assert ops.pending_device_error() == 0
        w.entries[1] = kept
    kept = w.ent_ptr.clone()
    w.ent_ptr[-1] = 1 << 30  # clamped to the entries there are
    assert torch.equal(ops.sparse_gated_linear(x, w, check=True), want)
    w.ent_ptr.copy_(kept)
    assert torch.equal(ops.sparse_gated_linear(x, w, check=True), want)


@pytest.mark.parametrize("tokens", [7, 50, 700])
def test_repeats_graphs_and_streams(tokens):
    x, dh, gate, up, wg, wu = case(tokens, 320, 320, 64, torch.bfloat16)
    w = ops.gated_weights(gate, up)

    def both(x, dh):
        return (ops.sparse_gated_linear(x, w), *ops.sparse_gated_linear_backward(dh, x, w))

    want = both(x, dh)
    assert all(torch.equal(a, b) for a, b in zip(want, both(x, dh)))
    other = [torch.randn_like(x), torch.randn_like(dh)]
    want2 = both(*other)
    # two graphs, captured on one stream, replayed at the same time
    inputs = [[x.clone(), dh.clone()] for _ in range(2)]
    graphs, outs, side = [], [], torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(x, dh)
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(both(*inputs[i]))
        graphs.append(g)
    for t, v in zip(inputs[1], other):
        t.copy_(v)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], want))
    assert all(torch.equal(a, b) for a, b in zip(outs[1], want2))
    # eager calls on two streams at once
    got = [None, None]
    for _ in range(3):
        for i, (args, s) in enumerate(zip(((x, dh), tuple(other)), streams)):
            with torch.cuda.stream(s):
                got[i] = both(*args)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got[0], want))
        assert all(torch.equal(a, b) for a, b in zip(got[1], want2))


def test_first_backward_in_a_capture_is_refused():
    x, dh, gate, up, wg, wu = case(8, 64, 64, 32, torch.bfloat16)
    w = ops.gated_weights(gate, up)
    ops.sparse_gated_linear(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(g, stream=s):
            ops.sparse_gated_linear_backward(dh, x, w)
    torch.cuda.synchronize()
    ops.sparse_gated_linear_backward(dh, x, w, check=True)


def test_offsets_beyond_32_bits():
    """H and dP of more than 2^32 values: the last tokens' rows are those of the same tokens alone."""
    tokens, m, k = 70_000, 32_768, 64
    x, dh, gate, up, wg, wu = case(130, m, k, 64, torch.bfloat16, keep=0.9)
    w = ops.gated_weights(gate, up)
    big = torch.zeros(tokens, k, device="cuda").bfloat16()
    big[-130:] = x
    h = ops.sparse_gated_linear(big, w, check=True)
    assert h.numel() > 2**31 and torch.equal(h[-130:], ops.sparse_gated_linear(x, w)) and not h[:-130].any()
    del h
    d = torch.zeros(tokens, m, device="cuda").bfloat16()
    d[-130:] = dh
    dx, db = ops.sparse_gated_linear_backward(d, big, w, check=True)
    dx1, db1 = ops.sparse_gated_linear_backward(dh, x, w)
    assert torch.equal(dx[-130:], dx1) and not dx[:-130].any()
    # the weight gradient adds the same 130 rows, in other steps of 16
    assert (db.double() - db1.double()).norm() <= torch.finfo(torch.bfloat16).eps * db1.double().norm()


def test_module_and_differences():
    """Gradients of the module against the formula's, and against differences of its own outputs."""
    x, dh, gate, up, wg, wu = case(60, 130, 100, 32, torch.float16, act="gelu_tanh", keep=0.6)
    layer = ops.SparseGatedLinear(gate, up, activation="gelu_tanh")
    xr = x.clone().requires_grad_(True)
    h = layer(xr)
    h.backward(dh)
    check(x, dh, wg, wu, gate, up, "gelu_tanh", h.detach(), xr.grad, *layer.weights().split(layer.blocks.grad))
    with torch.no_grad():
        assert torch.equal(layer(x), h)
    # along a direction: <dX, d> against (<dH, H(x + d)> - <dH, H(x - d)>) / 2.  H is rounded to fp16 and
    # its sums are off as above; beside that the difference of third order, taken from the formula.
    d = torch.randn_like(x) * 2.0**-5
    plus, minus = x + d, x - d
    delta = (plus.double() - minus.double()) / 2
    slope = (xr.grad.double() * delta).sum()
    with torch.no_grad():
        diff = ((layer(plus).double() - layer(minus).double()) * dh.double()).sum() / 2

    def exact(v):
        return act64(v.double() @ wg.t(), "gelu_tanh")[0] * (v.double() @ wu.t())

    true = ((exact(plus) - exact(minus)) * dh.double()).sum() / 2
    eps = torch.finfo(torch.float16).eps / 2
    noise = 2 * eps * ((exact(plus).abs() + exact(minus).abs()) * dh.double().abs()).sum() / 2
    assert (diff - true).abs() <= noise
    rounding = 4 * eps * ((xr.grad.double() * delta).abs()).sum() + noise
    f, da = act64(x.double() @ wg.t(), "gelu_tanh")
    grad64 = (dh.double() * (x.double() @ wu.t()) * da) @ wg + (dh.double() * f) @ wu
    curvature = (true - (grad64 * delta).sum()).abs()
    assert (slope - diff).abs() <= rounding + curvature


def test_module_patterns_may_be_loaded():
    """A state dict of another pattern with as many blocks: the kept structure follows."""
    pos = torch.tensor([0, 3, 5], device="cuda"), torch.tensor([1, 2, 6], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    mats = [weight(96, 96, 32, 0.3, torch.bfloat16, g, pos=p) for p in (*pos, pos[1], pos[0])]
    one = ops.SparseGatedLinear(mats[0][0], mats[1][0])
    two = ops.SparseGatedLinear(mats[2][0], mats[3][0])
    x, dh = torch.randn(9, 96, device="cuda").bfloat16(), torch.randn(9, 96, device="cuda").bfloat16()

    def grads(layer):
        layer.blocks.grad = None
        xr = x.clone().requires_grad_(True)
        layer(xr).backward(dh)
        return xr.grad, layer.blocks.grad.clone()

    grads(one)
    want = grads(two)
    one.load_state_dict(two.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(grads(one), want))
