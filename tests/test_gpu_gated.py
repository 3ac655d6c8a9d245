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

from kairo_b200 import ops
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


def check(x, dh, wg, wu, gate, up, act, h, dx, dgate, dup):
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
