"""Activations kept in 8 bits for the backward pass (CUDA only).

A layer that trains keeps its input for the weight gradient; in 8 bits it
takes 1.06 bytes a value instead of 2.  Every 64 columns of a row share a step
(the group's largest magnitude / 127), so that one loud column does not cost
the others their resolution:

* ``quantize_activations(X)`` -- the 8-bit codes and fp32 steps of X;
* ``dequantize_activations(q)`` -- what they stand for, in X's own type;
* ``sparse_linear_weight_grad(dY, q, W)`` and
  ``adapter_linear_backward(dY, q, ...)`` take them in X's place, and
  ``BlockSparseLinear(W, checkpoint="int8")`` keeps its input that way.

The reference has no counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor

from kairo_b200 import _lib

GROUP = 64  # columns that share a step


@dataclass(frozen=True)
class QuantizedActivations:
    """An (n, k) activation in 8 bits.

    codes: (n, k) int8, rows padded to 16 bytes (the last one too); steps:
    (ceil(k / 64), n) float32, the step of columns 64 g .. 64 g + 63 of row r at
    [g, r]; dtype: the activation's type, in which ``code * step`` is read
    back."""

    codes: Tensor
    steps: Tensor
    dtype: torch.dtype

    def __post_init__(self) -> None:
        if self.codes.dim() != 2 or self.codes.dtype != torch.int8:
            raise ValueError("codes must be a 2-D int8 tensor")
        n, k = self.codes.shape
        if self.steps.shape != ((k + GROUP - 1) // GROUP, n) or self.steps.dtype != torch.float32:
            raise ValueError(f"steps must be a ({(k + GROUP - 1) // GROUP}, {n}) float32 tensor")
        if self.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise TypeError(f"unsupported dtype {self.dtype}; expected float32, float16 or bfloat16")
        if self.steps.device != self.codes.device:
            raise ValueError("codes and steps must share a device")
        if n * k > 0:
            if self.codes.stride(1) != 1 or self.codes.data_ptr() % 16 or (n > 1 and (self.codes.stride(0) % 16 or
                                                                                    self.codes.stride(0) < k)):
                raise ValueError("codes must have 16-byte aligned rows")
            padded = -(-k // 16) * 16  # whole 16-byte vectors are read, of the last row too
            end = self.codes.storage_offset() + (n - 1) * self.codes.stride(0) + padded
            if end > self.codes.untyped_storage().nbytes():
                raise ValueError("codes must have rows padded to 16 bytes: the last row's memory ends before "
                                 f"column {padded}")
            if (n > 1 and self.steps.stride(1) != 1) or (self.steps.shape[0] > 1 and self.steps.stride(0) < n):
                raise ValueError("steps must be row-major")

    @classmethod
    def _made(cls, codes: Tensor, steps: Tensor, dtype: torch.dtype) -> "QuantizedActivations":
        """One whose parts this package laid out itself: no checks."""
        q = object.__new__(cls)
        q.__dict__.update(codes=codes, steps=steps, dtype=dtype)
        return q

    def _parts(self) -> tuple[Tensor, Tensor]:
        """Codes with the padding of their rows, and steps, for
        ``save_for_backward``: a copy of them (offloading hooks make some) keeps
        the padding, which a copy of ``codes`` does not."""
        n, k = self.codes.shape
        rows = self.codes if k % 16 == 0 else self.codes.as_strided((n, -(-k // 16) * 16), (self._ldq, 1))
        return rows, self.steps

    @classmethod
    def _from_parts(cls, rows: Tensor, steps: Tensor, k: int, dtype: torch.dtype) -> "QuantizedActivations":
        """The activation of k columns whose ``_parts()`` these are, or copies of them."""
        return cls(codes=rows[:, :k], steps=steps, dtype=dtype)

    @property
    def shape(self) -> tuple[int, int]:
        return tuple(self.codes.shape)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def is_cuda(self) -> bool:
        return self.codes.is_cuda

    @property
    def nbytes(self) -> int:
        """Bytes kept: codes with their row padding, and steps."""
        return self.shape[0] * self._ldq + 4 * self.steps.numel()

    @property
    def _ldq(self) -> int:
        n, k = self.codes.shape
        return self.codes.stride(0) if n > 1 and k > 0 else -(-k // 16) * 16

    @property
    def _lds(self) -> int:
        return self.steps.stride(0) if self.steps.shape[0] > 1 else self.steps.shape[1]


def quantize_activations(X: Tensor) -> QuantizedActivations:
    """X (n, k) float32, float16 or bfloat16 -> 8-bit codes and steps.

    A value is off by at most half a step, max|group| / 254.  A group whose
    largest magnitude is under 2^-100 reads back as zeros; one that holds an
    infinity or a NaN reads back as NaN."""
    index = _lib.device_index("quantize_activations", X)
    if X.dim() != 2:
        raise ValueError("X must be 2-D (n, k)")
    dt = _lib.kairo_dtype(X.dtype)
    if X.stride(1) != 1 or (X.shape[0] > 1 and X.stride(0) < X.shape[1]):
        X = X.contiguous()
    n, k = X.shape
    ldq = -(-k // 16) * 16
    if ldq == k or n == 0:
        codes = X.new_empty((n, k), dtype=torch.int8)
    else:  # rows padded to 16 bytes; room for the padding of the last
        codes = X.new_empty((n, ldq), dtype=torch.int8)[:, :k]
    steps = X.new_empty((-(-k // GROUP), n), dtype=torch.float32)
    _lib.launch("quantize_activations", _lib.lib().kairo_quantize_q8, index, X.data_ptr(), n, k, max(X.stride(0), k),
                dt, codes.data_ptr(), ldq, steps.data_ptr(), n)
    return QuantizedActivations._made(codes, steps, X.dtype)


def dequantize_activations(q: QuantizedActivations, *, out: Tensor | None = None) -> Tensor:
    """``code * step`` in the activation's type, (n, k)."""
    index = _lib.device_index("dequantize_activations", q.codes)
    n, k = q.shape
    if out is None:
        out = q.codes.new_empty((n, k), dtype=q.dtype)
    elif tuple(out.shape) != (n, k) or out.dtype != q.dtype or out.device != q.device or (
            k > 1 and out.stride(1) != 1) or (n > 1 and out.stride(0) < k):
        raise ValueError(f"out must be a row-major ({n}, {k}) {q.dtype} tensor on {q.device}")
    else:
        _lib.refuse_overlap("dequantize_activations", out, q.codes, q.steps)
    _lib.launch("dequantize_activations", _lib.lib().kairo_dequantize_q8, index, q.codes.data_ptr(), q._ldq,
                q.steps.data_ptr(), q._lds, n, k, out.data_ptr(), max(out.stride(0), k), _lib.kairo_dtype(q.dtype))
    return out
