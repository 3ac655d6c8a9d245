"""Cross entropy over a vocabulary: gradients by the losses of every size, finite or not."""

from __future__ import annotations

import pytest
import torch

from kairo_b200 import ops
from tests.test_gpu_vocab_loss import make, run_case, tiny, within

pytestmark = pytest.mark.gpu


def inputs(dtype, seed=0):
    """Values that are multiples of 2^-6 up to 2, and targets: products with powers of two are exact in fp16 and bf16."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def grid(*shape):
        return (torch.randint(-96, 97, shape, generator=g, device="cuda") / 64).to(dtype)

    return grid(50, 40), grid(300, 40), torch.randint(0, 300, (50,), generator=g, device="cuda"), g


def backward(x, w, ids, grad, scale=1.0):
    _, lse = ops.linear_cross_entropy(x, w, ids, scale=scale, reduction="none", return_lse=True, check=True)
    return ops.linear_cross_entropy_backward(grad, x, w, ids, lse, scale=scale, reduction="none", check=True)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_factor_that_is_not_finite(dtype, bad):
    """It reaches its own token's dX and the table's gradient, and no other token."""
    x, w, ids, g = inputs(dtype)
    grad = (torch.rand(50, generator=g, device="cuda") + 0.25) * 512
    dx, _ = backward(x, w, ids, torch.where(torch.arange(50, device="cuda") == 7, 0.0, grad))
    grad[7] = bad
    got, dw = backward(x, w, ids, grad)
    assert not torch.isfinite(got[7]).any() and not torch.isfinite(dw).all()
    others = torch.arange(50, device="cuda") != 7
    assert torch.equal(got[others], dx[others])


@pytest.mark.parametrize("dtype,powers", [(torch.float16, (-18, -9, 13)), (torch.bfloat16, (-60, -20, 20, 60))])
def test_factors_keep_their_digits(dtype, powers):
    """grad times 2^p gives the same digits: p is taken back by an operand times 2^p and a scale of 2^-p, which leave the logits as they are."""
    x, w, ids, g = inputs(dtype)
    grad = torch.rand(50, generator=g, device="cuda") + 0.25
    dx, dw = backward(x, w, ids, grad)
    assert dx.any() and dw.any()
    for p in powers:
        big = torch.tensor(2.0**p, dtype=torch.float64)
        up = (x.double() * big).to(dtype)
        assert torch.equal(up.double(), x.double() * big)  # exact
        got, _ = backward(up, w, ids, grad * 2.0**p, 2.0**-p)
        assert torch.equal(got, dx), p
        up = (w.double() * big).to(dtype)
        assert torch.equal(up.double(), w.double() * big)
        _, got = backward(x, up, ids, grad * 2.0**p, 2.0**-p)
        assert torch.equal(got, dw), p


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("tokens,vocab,dim", [(1, 1891, 256), (2, 1891, 250), (17, 700, 1024), (33, 5000, 130),
                                              (64, 257, 320), (100, 40000, 72), (128, 3001, 200)])
def test_few_tokens_are_rounded_once(tokens, vocab, dim, reduction, dtype):
    """Up to 128 tokens an entry of G over a 64th of its token's factor, and every target's, is held in two numbers: what
    stands in the results is their own rounding (h), h of the small entries, and the products' errors of 2^-13 as in
    test_gpu_vocab_loss; with G rounded once every target's h would stand there as well."""
    x, w, ids, g = make(tokens, vocab, dim, dtype, pad=0.0 if tokens < 5 else 0.1)
    grad = torch.rand(tokens, generator=g, device="cuda") + 0.5 if reduction == "none" else torch.tensor(0.7, device="cuda")
    loss, lse = ops.linear_cross_entropy(x, w, ids, reduction=reduction, return_lse=True, check=True)
    dx, dw = ops.linear_cross_entropy_backward(grad, x, w, ids, lse, reduction=reduction, check=True)
    live = (ids >= 0) & (ids < vocab)
    f = (grad.double() * live if reduction == "none" else grad.double() * live / live.sum().clamp(min=1))[:, None]
    xd, wd, at, h = x.double(), w.double(), ids.clamp(0, vocab - 1)[:, None], torch.finfo(dtype).eps / 2
    z = xd @ wd.t()
    lse64 = torch.logsumexp(z, 1)
    p = torch.exp(z - lse64[:, None])
    one = torch.zeros_like(p).scatter(1, at, 1.0)
    gd = (p - one) * f
    dz = (xd.abs() @ wd.abs().t()).amax(1) * 2.0**-17 + (lse64.abs() + 8) * 2.0**-21
    two = (one > 0) | (gd.abs() > f.abs() / 64 * 1.001)
    ga = gd.abs() * (torch.where(two, h * h, h) + 2.0**-13) + p * f.abs() * 2 * dz[:, None] + f.abs() * 2.0**-126
    if dtype == torch.float16:
        ga = ga + 2 * f.abs().max() * 2.0**-39  # of either number
    for name, got, want, tol in (("dX", dx, gd @ wd, ga @ wd.abs()), ("dW", dw, gd.t() @ xd, ga.t() @ xd.abs())):
        within(name, got, want, tol + (h + 2.0**-20) * want.abs() + tiny(dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_few_tokens_in_pieces(dtype):
    """A vocabulary of more than one piece for 128 tokens' two rows each; the last piece is narrow."""
    run_case(128, 1_048_576 + 300, 8, dtype, reduction="sum")
