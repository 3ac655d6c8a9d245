"""Embedding lookup with scaling, and its gradient by sorted tokens (CUDA only).

The dense-table counterpart of ``sparse_gather`` / ``sparse_scatter_grad``
(the reference's embedding path, kairo/ops/sparse_embedding.py:59-161, is
masked and wants a sorted unique id list):

* ``embedding_lookup(weight, ids, scale=s)`` -- ``s * weight[ids]``, computed
  in fp32 and rounded once.
* ``sort_tokens(ids, N)`` -- the token positions in id order (stable), for
  gradients of several tables or widths over one batch of ids.
* ``embedding_grad(grad_output, ids, N, scale=s)`` -- the (N, D) gradient,
  or the same added to an existing buffer (``out=..., accumulate=True``).
* ``ScaledEmbedding`` -- both as an autograd-aware module.

As in ``sparse_gather``, an id outside [0, N) gathers a zero row; it adds
nothing to the gradient.  A negative id therefore serves as padding.
"""

from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from kairo_b200 import _lib


def _flat_ids(ids: Tensor, op: str) -> Tensor:
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{op}: ids must be int32 or int64, got {ids.dtype}")
    if ids.dim() == 1 and ids.is_contiguous():
        return ids
    return ids.reshape(-1).contiguous()


def _rows(t: Tensor) -> Tensor:
    """``t`` (2-D) itself when its rows are contiguous and do not overlap."""
    if t.is_contiguous():
        return t
    n, d = t.shape
    return t if (d <= 1 or t.stride(1) == 1) and (n <= 1 or t.stride(0) >= d) else t.contiguous()


def _ld(t: Tensor) -> int:
    n, d = t.shape
    return max(t.stride(0), d) if n > 1 else d


@dataclass(frozen=True)
class TokenOrder:
    """Token positions in id order (``sort_tokens``).

    sorted_ids: (T,) int32, ids ascending, those outside [0, N) as N at the
    end; perm: (T,) int32, the token of every sorted position, ascending
    among equal ids; num_embeddings: N."""

    sorted_ids: Tensor
    perm: Tensor
    num_embeddings: int

    def __post_init__(self) -> None:
        for name, t in (("sorted_ids", self.sorted_ids), ("perm", self.perm)):
            if t.dim() != 1 or t.dtype != torch.int32 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous 1-D int32 tensor")
        if self.sorted_ids.shape != self.perm.shape or self.sorted_ids.device != self.perm.device:
            raise ValueError("sorted_ids and perm must be of one length, on one device")


@functools.lru_cache(maxsize=4096)
def _sort_bytes(tokens: int, n_rows: int) -> int:
    nbytes = ctypes.c_size_t(0)
    _lib.check(_lib.lib().kairo_token_sort_workspace_size(tokens, n_rows, ctypes.byref(nbytes)), "sort_tokens")
    return max(nbytes.value, 256)


@functools.lru_cache(maxsize=4096)
def _grad_bytes(tokens: int, dim: int, in_order: bool) -> int:
    nbytes = ctypes.c_size_t(0)
    _lib.check(_lib.lib().kairo_embedding_grad_workspace_size(tokens, dim, 1 if in_order else 0, ctypes.byref(nbytes)),
               "embedding_grad")
    return nbytes.value


def sort_tokens(ids: Tensor, num_embeddings: int) -> TokenOrder:
    """Stable order of the tokens ``ids`` (any shape, int32 or int64) by id, on the device."""
    index = _lib.device_index("sort_tokens", ids)
    n_rows = int(num_embeddings)
    if n_rows < 0:
        raise ValueError("num_embeddings must be non-negative")
    flat = _flat_ids(ids, "sort_tokens")
    n = flat.numel()
    out = flat.new_empty(n, dtype=torch.int32)
    perm = flat.new_empty(n, dtype=torch.int32)
    ws = flat.new_empty(_sort_bytes(n, n_rows), dtype=torch.uint8)
    _lib.launch("sort_tokens", _lib.lib().kairo_token_sort, index, flat.data_ptr(), flat.element_size(), n, n_rows,
                out.data_ptr(), perm.data_ptr(), ws.data_ptr(), ws.numel())
    return TokenOrder(sorted_ids=out, perm=perm, num_embeddings=n_rows)


def embedding_lookup(weight: Tensor, ids: Tensor, *, scale: float = 1.0, out_dtype: torch.dtype | None = None,
                     out: Tensor | None = None) -> Tensor:
    """``scale * weight[ids]``: ids.shape + (D,), in ``out_dtype`` (default: weight's), rounded once from fp32.

    weight: (N, D) float32, float16 or bfloat16; ids: int32 or int64, any
    shape; an id outside [0, N) gives a zero row.  ``out``: a contiguous
    tensor to write to."""
    index = _lib.device_index("embedding_lookup", weight, ids)
    if weight.dim() != 2 or weight.shape[1] < 1:
        raise ValueError("weight must be 2-D (N, D) with D >= 1")
    n, d = weight.shape
    flat = _flat_ids(ids, "embedding_lookup")
    in_dt = _lib.kairo_dtype(weight.dtype)
    odt = out_dtype or (out.dtype if out is not None else weight.dtype)
    out_dt = _lib.kairo_dtype(odt)
    shape = (*ids.shape, d)
    if out is None:
        out = weight.new_empty(shape) if odt == weight.dtype else weight.new_empty(shape, dtype=odt)
    elif tuple(out.shape) != shape or out.dtype != odt or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {shape} {odt} tensor")
    elif out.device != weight.device:
        raise ValueError("out must be on the weight's device")
    else:
        _lib.refuse_overlap("embedding_lookup", out, weight, flat)
    w = _rows(weight)
    _lib.launch("embedding_lookup", _lib.lib().kairo_embedding_lookup, index, w.data_ptr(), n, d, _ld(w), in_dt,
                flat.data_ptr(), flat.element_size(), flat.numel(), float(scale), out.data_ptr(), out_dt)
    return out


def embedding_grad(grad_output: Tensor, ids: Tensor | TokenOrder, num_embeddings: int, *, scale: float = 1.0,
                   out_dtype: torch.dtype | None = None, out: Tensor | None = None,
                   accumulate: bool = False) -> Tensor:
    """Gradient of ``embedding_lookup`` by its table: (N, D), row r = ``scale``
    times the sum of ``grad_output[t]`` over the tokens t with id r.

    grad_output: ids.shape + (D,); ids: the token ids or their
    ``sort_tokens(ids, N)``.  Sums are fp32 in an order fixed by the ids
    (deterministic, no atomics), rounded once to ``out_dtype`` (default:
    grad_output's).  With ``accumulate=True`` the sums are added to ``out``,
    whose other rows are neither read nor written; otherwise every row of
    ``out`` (or of a new tensor) is written."""
    n_rows = int(num_embeddings)
    if isinstance(ids, TokenOrder):
        if ids.num_embeddings != n_rows:
            raise ValueError(f"the token order is of {ids.num_embeddings} rows, not {n_rows}")
        tokens, where = ids.perm.numel(), (ids.perm, ids.sorted_ids)
    else:
        tokens, where = ids.numel(), (ids,)
    index = _lib.device_index("embedding_grad", grad_output, *where)
    dev = grad_output.device
    if n_rows < 0:
        raise ValueError("num_embeddings must be non-negative")
    if grad_output.dim() < 1 or grad_output.shape[-1] < 1:
        raise ValueError("grad_output must be (..., D) with D >= 1")
    d = grad_output.shape[-1]
    if not isinstance(ids, TokenOrder) and tuple(grad_output.shape[:-1]) != tuple(ids.shape):
        raise ValueError(f"grad_output must be {tuple(ids.shape) + (d,)}, got {tuple(grad_output.shape)}")
    g = _rows(grad_output if grad_output.dim() == 2 else grad_output.reshape(-1, d))
    if g.shape[0] != tokens:
        raise ValueError(f"grad_output has {g.shape[0]} rows for {tokens} tokens")
    odt = out_dtype or (out.dtype if out is not None else g.dtype)
    in_dt, out_dt = _lib.kairo_dtype(g.dtype), _lib.kairo_dtype(odt)
    if accumulate and out is None:
        raise ValueError("accumulate=True needs out")
    if out is None:
        out = g.new_empty((n_rows, d)) if odt == g.dtype else g.new_empty((n_rows, d), dtype=odt)
    elif tuple(out.shape) != (n_rows, d) or out.dtype != odt or out.device != dev or _rows(out) is not out:
        raise ValueError(f"out must be a row-major ({n_rows}, {d}) {odt} tensor on {dev}")
    else:
        _lib.refuse_overlap("embedding_grad", out, g, *where)
    in_order = isinstance(ids, TokenOrder)
    size = _grad_bytes(tokens, d, in_order)
    ws = g.new_empty(size, dtype=torch.uint8) if size else None
    tail = (tokens, n_rows, d, float(scale), out.data_ptr(), _ld(out), out_dt, 1 if accumulate else 0,
            ws.data_ptr() if size else None, size)
    if in_order:
        _lib.launch("embedding_grad", _lib.lib().kairo_embedding_grad_sorted, index, g.data_ptr(), _ld(g), in_dt,
                    ids.sorted_ids.data_ptr(), ids.perm.data_ptr(), *tail)
    else:
        flat = _flat_ids(ids, "embedding_grad")
        _lib.launch("embedding_grad", _lib.lib().kairo_embedding_grad, index, g.data_ptr(), _ld(g), in_dt,
                    flat.data_ptr(), flat.element_size(), *tail)
    return out


class _LookupFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight: Tensor, ids: Tensor, scale: float, out_dtype: torch.dtype | None) -> Tensor:
        ctx.save_for_backward(ids)
        ctx.rows, ctx.dtype, ctx.scale = weight.shape[0], weight.dtype, scale
        return embedding_lookup(weight, ids, scale=scale, out_dtype=out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):
        (ids,) = ctx.saved_tensors
        return embedding_grad(grad, ids, ctx.rows, scale=ctx.scale, out_dtype=ctx.dtype), None, None, None


class ScaledEmbedding(torch.nn.Module):
    """``scale * weight[ids]`` with the table's gradient from ``embedding_grad``.

    weight: (num_embeddings, embedding_dim), N(0, 1) initialised;
    ``out_dtype`` lets an fp32 table feed a 16-bit model."""

    def __init__(self, num_embeddings: int, embedding_dim: int, *, scale: float = 1.0,
                 dtype: torch.dtype = torch.float32, out_dtype: torch.dtype | None = None,
                 device: torch.device | str | None = None) -> None:
        super().__init__()
        if num_embeddings <= 0 or embedding_dim <= 0:
            raise ValueError("num_embeddings and embedding_dim must be positive")
        self.weight = torch.nn.Parameter(torch.randn(num_embeddings, embedding_dim, dtype=dtype, device=device))
        self.scale = float(scale)
        self.out_dtype = out_dtype

    def forward(self, ids: Tensor) -> Tensor:
        return _LookupFn.apply(self.weight, ids, self.scale, self.out_dtype)
