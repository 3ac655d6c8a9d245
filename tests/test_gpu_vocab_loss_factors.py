"""Cross entropy over a vocabulary: gradients by the losses of every size, finite or not."""

from __future__ import annotations

import pytest
import torch

from kairo_b200 import ops

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
