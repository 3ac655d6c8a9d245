"""Softmax cross entropy against a whole vocabulary, without keeping the logits (CUDA only).

The loss that trains a model whose tokens come in through ``embedding_lookup``:
its table (or another of the same kind) scores every token of the vocabulary,

    z[t, v] = scale * X[t] . weight[v]      lse[t] = log sum_v exp z[t, v]
    loss[t] = lse[t] - z[t, targets[t]]

* ``linear_cross_entropy`` -- the loss and lse; ``-loss`` is a token's
  log-probability, so this also scores tokens when serving.
* ``linear_cross_entropy_backward`` -- the gradients by X and weight.
* ``LinearCrossEntropy`` -- both as a module with autograd, on a table of its
  own or on a ``ScaledEmbedding``'s.

The tokens x vocabulary logits are never in memory: the forward pass keeps 8
bytes per token and 128 tokens of the vocabulary, the backward pass forms the
logits again in pieces of the vocabulary.  As in ``embedding_lookup``, where an
id outside [0, N) gathers a zero row, a target outside [0, V), such as -1 or
-100 for padding, counts for nothing: its loss is 0, it gives no gradient, and
``reduction="mean"`` divides by the others.

The reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from kairo_b200 import _lib
from kairo_b200.ops.token_embedding import ScaledEmbedding, _flat_ids, _ld, _rows

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _problem(op: str, X: Tensor, weight: Tensor, targets: Tensor, reduction: str):
    """Checked (X as rows, weight as rows, flat targets, tokens, vocab, dim, dtype code, reduction code)."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{op}: reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"{op}: weight must be (V, D) with V and D >= 1, got {tuple(weight.shape)}")
    v, d = weight.shape
    if X.dim() < 1 or X.shape[-1] != d or X.shape[:-1] != targets.shape:
        raise ValueError(f"{op}: X must be targets.shape + ({d},), got {tuple(X.shape)} and targets "
                         f"{tuple(targets.shape)}")
    if X.dtype != weight.dtype:
        raise TypeError(f"{op}: X is {X.dtype}, weight is {weight.dtype}")
    if X.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"{op}: X and weight must be float16 or bfloat16, got {X.dtype}")
    ids = _flat_ids(targets, op)
    return (_rows(X if X.dim() == 2 else X.reshape(-1, d)), _rows(weight), ids, ids.numel(), v, d,
            _lib.kairo_dtype(X.dtype), _REDUCTIONS[reduction])


def _aligned(t: Tensor | None) -> tuple[int, int]:
    """An address and a row pitch that are as 16-byte aligned as ``t``'s rows: all that workspace sizes depend on."""
    if t is None:
        return 0, 0
    return 16 + t.data_ptr() % 16, _ld(t) % 8


@functools.lru_cache(maxsize=4096)
def _forward_bytes(x: tuple[int, int], w: tuple[int, int], tokens: int, v: int, d: int) -> int:
    nbytes, up = ctypes.c_size_t(0), -(-d // 8) * 8
    _lib.check(_lib.lib().kairo_vocab_loss_workspace_size(x[0], up + x[1], w[0], up + w[1], tokens, v, d,
                                                          ctypes.byref(nbytes)), "linear_cross_entropy")
    return nbytes.value


@functools.lru_cache(maxsize=4096)
def _backward_bytes(w: tuple[int, int], dx: tuple[int, int], dw: tuple[int, int], tokens: int, v: int, d: int) -> int:
    nbytes, up = ctypes.c_size_t(0), -(-d // 8) * 8
    _lib.check(_lib.lib().kairo_vocab_loss_backward_workspace_size(
        w[0], up + w[1], tokens, v, d, dx[0] or None, up + dx[1], dw[0] or None, up + dw[1], ctypes.byref(nbytes)),
        "linear_cross_entropy_backward")
    return nbytes.value


def linear_cross_entropy(X: Tensor, weight: Tensor, targets: Tensor, *, scale: float = 1.0, reduction: str = "mean",
                         return_lse: bool = False, check: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """Cross entropy of ``targets`` under the logits ``scale * X @ weight^T``, in float32.

    X: targets.shape + (D,), weight: (V, D), both float16 or both bfloat16;
    targets: int32 or int64, one outside [0, V) counts for nothing.
    ``reduction``: "none" (targets' shape), "sum", or "mean" over the targets
    that count (0 without any).  ``return_lse=True`` also returns lse (targets'
    shape, float32), which ``linear_cross_entropy_backward`` takes.

    ``check=True`` synchronises and raises KairoDeviceError where a kernel's
    wait ran out; without it ``pending_device_error`` tells."""
    op = "linear_cross_entropy"
    index = _lib.device_index(op, X, weight, targets)
    x, w, ids, tokens, v, d, dt, red = _problem(op, X, weight, targets, reduction)
    shape = targets.shape
    lse = x.new_empty(shape, dtype=torch.float32)
    loss = x.new_empty(shape if reduction == "none" else (), dtype=torch.float32)
    ws = x.new_empty(_forward_bytes(_aligned(x), _aligned(w), tokens, v, d), dtype=torch.uint8)
    err = _lib.error_word(index)
    if check:
        _lib.take_pending_error(err, op)
    _lib.launch(op, _lib.lib().kairo_vocab_loss, index, x.data_ptr(), _ld(x), w.data_ptr(), _ld(w), tokens, v, d, dt,
                ids.data_ptr(), ids.element_size(), float(scale), red, loss.data_ptr(), lse.data_ptr(), ws.data_ptr(),
                ws.numel(), err.data_ptr())
    if check:
        _lib.raise_on_device_error(err)
    return (loss, lse) if return_lse else loss


def _gradient(op: str, name: str, out: Tensor | None, like: Tensor, rows: int, d: int, *inputs: Tensor) -> Tensor:
    if out is None:
        return like.new_empty((rows, d))
    if out.shape != (rows, d) or out.dtype != like.dtype or out.device != like.device or _rows(out) is not out:
        raise ValueError(f"{op}: {name} must be a row-major ({rows}, {d}) {like.dtype} tensor on {like.device}")
    _lib.refuse_overlap(op, out, *inputs)
    return out


def linear_cross_entropy_backward(grad: Tensor, X: Tensor, weight: Tensor, targets: Tensor, lse: Tensor, *,
                                  scale: float = 1.0, reduction: str = "mean", need_dx: bool = True,
                                  need_dw: bool = True, dw: Tensor | None = None, check: bool = False
                                  ) -> tuple[Tensor | None, Tensor | None]:
    """(dX, d_weight) of ``linear_cross_entropy``, in X's type, shaped like X and weight.

    grad: the gradient by the loss, float32: one number, or targets' shape for
    ``reduction="none"``; lse: what ``return_lse`` gave.  Either result may be
    left out (None).  ``dw``: a row-major (V, D) tensor for d_weight; every row
    is written.

    A token that does not count has a dX of zeros and does not enter d_weight,
    whatever its X and lse hold."""
    op = "linear_cross_entropy_backward"
    index = _lib.device_index(op, X, weight, targets, grad, lse)
    x, w, ids, tokens, v, d, dt, red = _problem(op, X, weight, targets, reduction)
    each = reduction == "none"
    if grad.dtype != torch.float32 or (grad.shape != targets.shape if each else grad.numel() != 1):
        raise ValueError(f"{op}: grad must be float32, {'of the shape of the targets' if each else 'one number'}; got "
                         f"{tuple(grad.shape)} {grad.dtype}")
    if lse.dtype != torch.float32 or lse.shape != targets.shape:
        raise ValueError(f"{op}: lse must be float32, of the shape of the targets; got {tuple(lse.shape)} {lse.dtype}")
    grad, lse = grad.contiguous(), lse.contiguous()
    dX = x.new_empty((tokens, d)) if need_dx else None
    if need_dw:
        dw = _gradient(op, "dw", dw, w, v, d, x, w, ids, grad, lse)
    elif dw is not None:
        raise ValueError(f"{op}: dw is given and need_dw is False")
    if need_dx or need_dw:
        results = (_lib.ptr(dX), d, _lib.ptr(dw), d if dw is None else _ld(dw))
        ws = x.new_empty(_backward_bytes(_aligned(w), _aligned(dX), _aligned(dw), tokens, v, d), dtype=torch.uint8)
        err = _lib.error_word(index)
        if check:
            _lib.take_pending_error(err, op)
        _lib.launch(op, _lib.lib().kairo_vocab_loss_backward, index, grad.data_ptr(), x.data_ptr(), _ld(x),
                    w.data_ptr(), _ld(w), tokens, v, d, dt, ids.data_ptr(), ids.element_size(), float(scale), red,
                    lse.data_ptr(), *results, ws.data_ptr(), ws.numel(), err.data_ptr())
        if check:
            _lib.raise_on_device_error(err)
    return dX if dX is None else dX.view(X.shape), dw


class _CrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X: Tensor, weight: Tensor, targets: Tensor, scale: float, reduction: str) -> Tensor:
        loss, lse = linear_cross_entropy(X, weight, targets, scale=scale, reduction=reduction, return_lse=True)
        ctx.save_for_backward(X, weight, targets, lse)
        ctx.how = {"scale": scale, "reduction": reduction}
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):
        X, weight, targets, lse = ctx.saved_tensors
        dX, dw = linear_cross_entropy_backward(grad, X, weight, targets, lse, need_dx=ctx.needs_input_grad[0],
                                               need_dw=ctx.needs_input_grad[1], **ctx.how)
        return dX, dw, None, None, None


class LinearCrossEntropy(torch.nn.Module):
    """``linear_cross_entropy`` with autograd: ``forward(X, targets)``.

    table: the (V, D) parameter that scores the vocabulary, or the
    ``ScaledEmbedding`` whose table does (tied weights: its gradient is the sum
    of the lookup's and the loss's)."""

    def __init__(self, table: torch.nn.Parameter | ScaledEmbedding, *, scale: float = 1.0,
                 reduction: str = "mean") -> None:
        super().__init__()
        weight = table.weight if isinstance(table, ScaledEmbedding) else table
        if not isinstance(weight, torch.nn.Parameter) or weight.dim() != 2:
            raise TypeError("table must be a (V, D) Parameter or a ScaledEmbedding")
        if weight.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"the table must be float16 or bfloat16, got {weight.dtype}")
        if reduction not in _REDUCTIONS:
            raise ValueError(f"reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
        self.weight = weight
        self.scale = float(scale)
        self.reduction = reduction

    def forward(self, X: Tensor, targets: Tensor) -> Tensor:
        return _CrossEntropyFn.apply(X, self.weight, targets, self.scale, self.reduction)
