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
