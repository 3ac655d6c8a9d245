"""Cross entropy over a vocabulary table and its gradients, against the formulas in 64 bits.

Bounds.  A logit z is a sum of dim products added 16 at a time; in segments of
256 each step is off by at most 2^-22 of the sum's absolute terms A (16 steps),
their sums by 2^-24 a segment: under A * 2^-17 for the widths here.  exp2 is off
by 2^-22 of its value and by 2^-23 |z| through its argument.  So lse, a weighted
mean of the logits' errors, is off by at most A * 2^-17 + (|lse| + 8) * 2^-21, and the
loss by the sum of two such.  G is rounded to 16 bits once, h = eps / 2 of each
entry, beside the error dz of its exponent; its products add 2^-14 of their
absolute terms, and the result is rounded again.
"""

from __future__ import annotations

import math

import pytest
import torch

from kairo_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def make(tokens, vocab, dim, dtype, seed=0, pad=0.1, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(vocab, dim, generator=g, device="cuda") * spread * dim**-0.5).to(dtype)
    ids = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
    x = (torch.randn(tokens, dim, generator=g, device="cuda") + w[ids].float()).to(dtype)
    drop = torch.rand(tokens, generator=g, device="cuda") < pad
    return x, w, torch.where(drop, torch.where(ids % 2 == 0, -1, vocab + 5), ids), g


def reference(x, w, ids, scale, grad, reduction):
    """Losses, lse, dX, dW and the bounds of each, in 64 bits."""
    h = torch.finfo(x.dtype).eps / 2
    vocab = w.shape[0]
    live = (ids >= 0) & (ids < vocab)
    xd, wd = torch.where(live[:, None], x.double(), 0.0), w.double()
    xa = x.double()
    z = scale * (xa @ wd.t())
    a = abs(scale) * (xa.abs() @ wd.abs().t()).amax(1)  # absolute terms of a logit, the row's largest
    lse = torch.logsumexp(z, 1)
    at = ids.clamp(0, vocab - 1)[:, None]
    each = torch.where(live, lse - z.gather(1, at)[:, 0], 0.0)
    dz = a * 2.0**-17 + (lse.abs() + 8) * 2.0**-21
    count = max(1, int(live.sum()))
    f = {"none": grad.double(), "sum": grad.double().expand(len(ids)),
         "mean": grad.double().expand(len(ids)) / count}[reduction] * live
    p = torch.exp(z - lse[:, None])
    g = (p.scatter_add(1, at, torch.full_like(at, -1.0, dtype=torch.float64))) * f[:, None]
    g = torch.where(live[:, None], g, 0.0)
    ga = g.abs() * (h + 2.0**-13) + torch.where(live[:, None], p * f.abs()[:, None] * 2 * dz[:, None], 0.0)
    # exp2 gives 0 for results under fp32's smallest normal number, so an entry may lack up to 2^-126 of its factor
    ga = ga + f.abs()[:, None] * 2.0**-126
    if x.dtype == torch.float16:  # entries under fp16's smallest step, after the lift by 2^15 and the factors' power of two
        ga = ga + f.abs().max() * 2.0**-39
    dx, dw = scale * (g @ wd), scale * (g.t() @ xd)
    tol_x = abs(scale) * (ga @ wd.abs()) + (h + 2.0**-20) * dx.abs() + tiny(x.dtype)
    tol_w = abs(scale) * (ga.t() @ xd.abs()) + (h + 2.0**-20) * dw.abs() + tiny(x.dtype)
    loss = {"none": each, "sum": each.sum(), "mean": each.sum() / count}[reduction]
    tol = torch.where(live, 2 * dz, 0.0) + 2.0**-22 * each.abs()
    tol_loss = {"none": tol, "sum": tol.sum() + each.sum() * 2.0**-20,
                "mean": tol.sum() / count + each.sum() / count * 2.0**-20}[reduction]
    return loss, tol_loss, lse, dz, dx, tol_x, dw, tol_w


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2  # half of the smallest step


def within(name, got, want, tol):
    off = (got.double() - want).abs() - tol
    assert torch.isfinite(got.double()).all(), f"{name} is not finite"
    worst = off.max() if off.numel() else torch.tensor(-1.0)
    assert worst <= 0, f"{name}: {worst.item():.3g} over its bound"


def run_case(tokens, vocab, dim, dtype, *, scale=1.0, reduction="mean", pad=0.1, seed=0, spread=2.0):
    x, w, ids, g = make(tokens, vocab, dim, dtype, seed, pad, spread)
    grad = torch.randn(tokens if reduction == "none" else (), generator=g, device="cuda")
    loss, tol, lse, dz, dx, tol_x, dw, tol_w = reference(x, w, ids, scale, grad, reduction)
    got, got_lse = ops.linear_cross_entropy(x, w, ids, scale=scale, reduction=reduction, return_lse=True, check=True)
    assert got.dtype == got_lse.dtype == torch.float32 and got.shape == loss.shape
    within("lse", got_lse, lse, dz)
    within("loss", got, loss, tol)
    gx, gw = ops.linear_cross_entropy_backward(grad, x, w, ids, got_lse, scale=scale, reduction=reduction, check=True)
    assert gx.dtype == gw.dtype == dtype and gx.shape == x.shape and gw.shape == w.shape
    within("dX", gx, dx, tol_x)
    within("dW", gw, dw, tol_w)
    return x, w, ids, got, got_lse, gx, gw, grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,vocab,dim", [(4, 300, 64), (1, 1, 8), (1, 257, 64), (2, 256, 65), (127, 255, 63),
                                              (128, 1000, 128), (129, 129, 200), (257, 4099, 64), (300, 513, 1001),
                                              (513, 2, 1), (33, 70000, 7), (1000, 3001, 512)])
def test_sizes(tokens, vocab, dim, dtype):
    run_case(tokens, vocab, dim, dtype)


@pytest.mark.parametrize("tokens,vocab,dim", [(40, 1, 1001), (200, 1, 33), (1, 1, 5), (1, 300, 1001), (200, 2, 999)])
def test_single_rows(tokens, vocab, dim):
    """A table or a batch of one row whose width is no multiple of 8."""
    run_case(tokens, vocab, dim, torch.bfloat16, pad=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("scale", [1.0, -0.7, 3.0, 0.0])
def test_reductions_and_scales(reduction, scale, dtype):
    run_case(70, 700, 96, dtype, reduction=reduction, scale=scale)


@pytest.mark.parametrize("tokens", [5, 15, 16, 64, 65, 128, 300])
def test_token_counts(tokens):
    """Copies of few tokens, 64 rows of the row operand, one row of tiles, several."""
    run_case(tokens, 1500, 320, torch.bfloat16, reduction="none")


@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces(dtype):
    """More logits than one piece of the backward pass holds; the last piece is narrower."""
    run_case(4100, 70001, 64, dtype, pad=0.05)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spread,scale", [(40.0, 1.0), (2.0, 100.0), (0.01, 1.0)])
def test_steep_and_flat(spread, scale, dtype):
    """Logits of hundreds, where a token takes nearly all of the sum, and logits that are nearly alike."""
    run_case(140, 900, 64, dtype, spread=spread, scale=scale)


def test_weighted_tokens_of_any_size():
    """Factors from 2^-60 to 2^60 keep their digits in fp16, as the shared power of two goes by the largest."""
    for size in (2.0**-60, 2.0**60):
        x, w, ids, g = make(50, 300, 40, torch.float16, pad=0.0)
        grad = torch.rand(50, generator=g, device="cuda")
        _, lse = ops.linear_cross_entropy(x, w, ids, reduction="none", return_lse=True)
        dx, dw = ops.linear_cross_entropy_backward(grad, x, w, ids, lse, reduction="none")
        # a power of two in the gradient and its inverse in the scale give the same sums
        dx2, dw2 = ops.linear_cross_entropy_backward(grad * size, x, w, ids, lse, reduction="none")
        big = size > 1
        assert torch.equal(torch.isinf(dx2).any(), torch.tensor(big, device="cuda")) or not big
        if not big:
            assert not dx2.any() and not dw2.any()  # under fp16's smallest step
    assert dx.any() and dw.any()


def test_layouts():
    x, w, ids, g = make(130, 601, 120, torch.bfloat16)
    grad = torch.randn((), generator=g, device="cuda")
    loss, lse = ops.linear_cross_entropy(x, w, ids, return_lse=True)
    dx, dw = ops.linear_cross_entropy_backward(grad, x, w, ids, lse)

    def same(x2, w2, ids2, shape=(130,)):
        l2, s2 = ops.linear_cross_entropy(x2, w2, ids2, return_lse=True)
        assert torch.equal(l2, loss) and s2.shape == shape and torch.equal(s2.reshape(-1), lse)
        a, b = ops.linear_cross_entropy_backward(grad, x2, w2, ids2, s2)
        assert a.shape == x2.shape and torch.equal(a.reshape(dx.shape), dx) and torch.equal(b, dw)

    same(x.view(10, 13, 120), w, ids.view(10, 13), (10, 13))
    same(x, w, ids.int())
    same(x.t().contiguous().t(), w.t().contiguous().t(), ids)
    same(x, w, torch.stack([ids, ids], 1)[:, 0])
    for at in (0, 8, 1, 5):
        wx, ww = torch.full((130, 200), 3.0, device="cuda").bfloat16(), torch.full((601, 168), 3.0, device="cuda").bfloat16()
        wx[:, at:at + 120], ww[:, at:at + 120] = x, w
        same(wx[:, at:at + 120], ww[:, at:at + 120], ids)
        out = torch.full((603, 200), 4.0, device="cuda").bfloat16()
        view = out[1:602, at:at + 120]
        got = ops.linear_cross_entropy_backward(grad, x, w, ids, lse, need_dx=False, dw=view)
        assert got[0] is None and got[1] is view and torch.equal(view, dw)
        out[1:602, at:at + 120] = 4
        assert (out == 4).all()  # nothing around the result was written
    assert ops.linear_cross_entropy_backward(grad, x, w, ids, lse, need_dw=False)[1] is None


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_nothing_counts(reduction):
    x, w, ids, g = make(40, 300, 64, torch.bfloat16)
    x[3], x[4] = float("nan"), float("inf")
    none = torch.full_like(ids, -100)
    loss, lse = ops.linear_cross_entropy(x, w, none, reduction=reduction, return_lse=True)
    assert not loss.any() and (loss.shape == (40,) if reduction == "none" else loss.shape == ())
    grad = torch.ones_like(loss)
    dx, dw = ops.linear_cross_entropy_backward(grad, x, w, none, lse, reduction=reduction)
    assert not dx.any() and not dw.any()
    # no tokens at all
    loss, lse = ops.linear_cross_entropy(x[:0], w, ids[:0], reduction=reduction, return_lse=True)
    assert not loss.any() and lse.numel() == 0
    dx, dw = ops.linear_cross_entropy_backward(torch.ones_like(loss), x[:0], w, ids[:0], lse, reduction=reduction)
    assert dx.shape == (0, 64) and dw.shape == w.shape and not dw.any()


def test_not_finite():
    """What a padded token holds reaches nothing; what a counted one holds reaches its own loss and gradient."""
    x, w, ids, g = make(300, 500, 72, torch.bfloat16, pad=0.0)
    ids[[5, 200]] = -1
    kw = {"reduction": "none"}
    grad = torch.randn(300, generator=g, device="cuda")
    loss, lse = ops.linear_cross_entropy(x, w, ids, return_lse=True, **kw)
    want = ops.linear_cross_entropy_backward(grad, x, w, ids, lse, **kw)
    bad = x.clone()
    bad[5], bad[200, 3] = float("nan"), float("-inf")
    loss2, lse2 = ops.linear_cross_entropy(bad, w, ids, return_lse=True, **kw)
    assert torch.equal(loss2, loss)
    got = ops.linear_cross_entropy_backward(grad, bad, w, ids, lse2, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    bad = x.clone()
    bad[7, 0] = float("inf")
    loss3, _ = ops.linear_cross_entropy(bad, w, ids, return_lse=True, **kw)
    assert not torch.isfinite(loss3[7])
    keep = torch.arange(300, device="cuda") != 7
    assert torch.equal(loss3[keep], loss[keep])
    got = ops.linear_cross_entropy_backward(grad, bad, w, ids, lse.where(keep, torch.nan), **kw)
    assert torch.equal(got[0][keep], want[0][keep]) and not torch.isfinite(got[0][7]).any()
    # a logit of minus infinity has no probability; a table row that is all of it gives its targets an infinite loss
    low = w.clone()
    low[9] = 0
    low[9, 0] = float("-inf")
    pos = x.abs()
    l, s = ops.linear_cross_entropy(pos, low, torch.full_like(ids, 9), return_lse=True, **kw)
    assert torch.isfinite(s).all() and (l == float("inf")).all()


def test_repeats_graphs_and_streams():
    x, w, ids, g = make(300, 5000, 200, torch.bfloat16)
    grad = torch.randn(300, generator=g, device="cuda")

    def both(x, ids):
        loss, lse = ops.linear_cross_entropy(x, w, ids, reduction="none", return_lse=True)
        mean = ops.linear_cross_entropy(x, w, ids)
        return (loss, lse, mean, *ops.linear_cross_entropy_backward(grad, x, w, ids, lse, reduction="none"))

    want = both(x, ids)
    assert all(torch.equal(a, b) for a, b in zip(want, both(x, ids)))
    other = [torch.randn_like(x), ids.flip(0).clone()]
    want2 = both(*other)
    inputs = [[x.clone(), ids.clone()] for _ in range(2)]
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(both(*inputs[i]))
        graphs.append(gr)
    for t, v in zip(inputs[1], other):
        t.copy_(v)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], want))
    assert all(torch.equal(a, b) for a, b in zip(outs[1], want2))
    got = [None, None]
    for _ in range(3):
        for i, (args, s) in enumerate(zip(((x, ids), tuple(other)), streams)):
            with torch.cuda.stream(s):
                got[i] = both(*args)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got[0], want))
        assert all(torch.equal(a, b) for a, b in zip(got[1], want2))
    assert ops.pending_device_error() == 0


def test_offsets_beyond_32_bits():
    """A table of more than 2^31 values: targets in its last rows."""
    vocab, dim = 530_000, 4096
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.empty(vocab, dim, dtype=torch.bfloat16, device="cuda").normal_(0, 2 * dim**-0.5, generator=g)
    ids = torch.tensor([vocab - 1, 0, vocab - 300, 17], device="cuda")
    x = (torch.randn(4, dim, generator=g, device="cuda") + w[ids].float()).bfloat16()
    assert w.numel() > 2**31
    z = torch.cat([x.double() @ c.double().t() for c in w.split(50_000)], 1)
    lse = torch.logsumexp(z, 1)
    a = torch.stack([(x.double().abs() @ c.double().abs().t()).amax(1) for c in w.split(50_000)]).amax(0)
    dz = a * 2.0**-17 + (lse + 8) * 2.0**-21
    loss, s = ops.linear_cross_entropy(x, w, ids, reduction="none", return_lse=True, check=True)
    within("lse", s, lse, dz)
    within("loss", loss, lse - z.gather(1, ids[:, None])[:, 0], 2 * dz)
    grad = torch.ones(4, device="cuda")
    dx, dw = ops.linear_cross_entropy_backward(grad, x, w, ids, s, reduction="none", check=True)
    p = torch.exp(z - lse[:, None]).scatter_add(1, ids[:, None], torch.full((4, 1), -1.0, dtype=torch.float64, device="cuda"))
    for rows in (slice(0, 40), slice(vocab - 400, vocab)):
        want = p[:, rows].t() @ x.double()
        assert (dw[rows].double() - want).norm() <= 2 * torch.finfo(torch.bfloat16).eps * want.norm()
    want = sum(p[:, i:i + 50_000] @ w[i:i + 50_000].double() for i in range(0, vocab, 50_000))
    assert (dx.double() - want).norm() <= 2 * torch.finfo(torch.bfloat16).eps * want.norm()


def test_module_and_differences():
    """Gradients through autograd, and against differences of the loss itself."""
    x, w, ids, g = make(200, 700, 96, torch.float16)
    table = torch.nn.Parameter(w.clone())
    layer = ops.LinearCrossEntropy(table, scale=0.8, reduction="sum")
    xr = x.clone().requires_grad_(True)
    layer(xr, ids).backward()
    one = torch.ones((), device="cuda")
    _, _, _, _, dx, tol_x, dw, tol_w = reference(x, w, ids, 0.8, one, "sum")
    within("dX", xr.grad, dx, tol_x)
    within("dW", table.grad, dw, tol_w)

    def loss_at(v, t):
        loss, tol, *_ = reference(v, t, ids, 0.8, one, "sum")
        return ops.linear_cross_entropy(v, t, ids, scale=0.8, reduction="sum").double(), loss, tol

    for which, at, grad, true, tol in (("x", x, xr.grad, dx, tol_x), ("w", w, table.grad, dw, tol_w)):
        d = torch.randn(at.shape, generator=g, device="cuda").half() * 2.0**-6
        plus, minus = at + d, at - d
        delta = (plus.double() - minus.double()) / 2
        (lp, ep, tp), (lm, em, tm) = (loss_at(v, w) if which == "x" else loss_at(x, v) for v in (plus, minus))
        curvature = ((ep - em) / 2 - (true * delta).sum()).abs()  # of third order, from the formula
        off = ((lp - lm) / 2 - (grad.double() * delta).sum()).abs()
        assert off <= (tp + tm) / 2 + (tol * delta.abs()).sum() + curvature


def test_tied_model_step():
    """Ids through the scaled embedding, a block-sparse feed-forward block beside a skip connection and the loss over
    the same table: every gradient against the dense model in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(11)
    vocab, dim, wide, tokens = 900, 192, 320, 333
    emb = ops.ScaledEmbedding(vocab, dim, scale=dim**0.5, dtype=torch.bfloat16, device="cuda")
    with torch.no_grad():
        emb.weight.copy_(torch.randn(vocab, dim, generator=g, device="cuda") * dim**-0.5)
    mats, dense = [], []
    for m, k in ((wide, dim), (wide, dim), (dim, wide)):
        nbr, nbc = -(-m // 64), -(-k // 64)
        pos = torch.nonzero(torch.rand(nbr * nbc, generator=g, device="cuda") < 0.6)[:, 0]
        blocks = (torch.randn(pos.numel(), 64, 64, generator=g, device="cuda") * (0.6 * k) ** -0.5).bfloat16()
        mats.append(ops.bsr_from_tiles(blocks, (pos // nbc).int(), (pos % nbc).int(), (m, k)))
        dense.append((blocks, pos, nbr, nbc, m, k))
    ffn = ops.SparseFeedForward(*mats, activation="silu")
    head = ops.LinearCrossEntropy(emb)
    ids = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
    targets = torch.where(torch.rand(tokens, generator=g, device="cuda") < 0.1, -1, ids.roll(-1))
    x = emb(ids)
    loss = head(x + ffn(x), targets)
    loss.backward()

    table = emb.weight.detach().double().requires_grad_(True)
    blocks = [d[0].double().requires_grad_(True) for d in dense]

    def full(b, pos, nbr, nbc, m, k):
        out = torch.zeros(nbr, nbc, 64, 64, dtype=torch.float64, device="cuda").index_put((pos // nbc, pos % nbc), b)
        return out.transpose(1, 2).reshape(nbr * 64, nbc * 64)[:m, :k]

    wg, wu, wd = (full(b, *d[1:]) for b, d in zip(blocks, dense))
    xe = table[ids] * dim**0.5
    y = xe + (torch.nn.functional.silu(xe @ wg.t()) * (xe @ wu.t())) @ wd.t()
    ref = torch.nn.functional.cross_entropy(y @ table.t(), targets, ignore_index=-1)
    ref.backward()
    # x, H, the block's output, x + it and the gradients on the way back are rounded to bf16, about ten roundings of
    # eps / 2 of their values one after the other; as 2-norms they add up to less than ten times that.
    bound = 10 * torch.finfo(torch.bfloat16).eps / 2
    assert (loss.double() - ref).abs() <= bound * ref
    dgate, dup = ffn.gated.weights().split(ffn.gated.blocks.grad)
    for name, got, want in (("table", emb.weight.grad, table.grad), ("gate", dgate, blocks[0].grad),
                            ("up", dup, blocks[1].grad), ("down", ffn.down.blocks.grad, blocks[2].grad)):
        off = (got.double() - want).norm() / want.norm()
        assert off <= bound, f"{name}: {off.item():.3g}"
