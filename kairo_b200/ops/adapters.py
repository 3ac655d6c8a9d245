"""Low-rank adapters of many requests in one batch, beside a shared
projection (CUDA only).

Every token of a batch may name one of G adapters (a rank-R correction of the
projection's weight) or none:

    low[t] = scale[a] * X[t] down[a]^T        Y[t] = base[t] + low[t] up[a]

``base`` is the shared projection's output (``sparse_linear`` or any other).
``up`` is stored rank row by rank row like ``down`` -- (G, R, out_features),
the transpose of the usual (out_features, R) -- so that the backward pass is
the same kernel with the two swapped.

* ``adapter_plan(ids, G)`` -- the batch's tokens ordered by adapter, on the
  device; made once per batch, used by every layer.
* ``adapter_linear`` -- Y, for single tokens and prompts alike.
* ``adapter_linear_backward`` -- dX and the gradients of down and up.
* ``adapted_sparse_linear`` -- ``sparse_linear`` and the adapters, summed in
  fp32 and rounded once.
* ``AdaptedSparseLinear`` -- the same as a module with autograd.

The reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from kairo_b200 import _lib
from kairo_b200.ops.backward import (
    BlockSparseLinear,
    sparse_linear_weight_grad,
    transpose_values,
)
from kairo_b200.ops.checkpoint import QuantizedActivations, quantize_activations
from kairo_b200.ops.spmm import KernelConfig, sparse_linear
from kairo_b200.ops.token_embedding import _flat_ids, _ld, _rows
from kairo_b200.types import BlockSparseMatrix

MAX_RANK = 128


@dataclass(frozen=True)
class LowRankAdapters:
    """G adapters of one projection.

    down: (G, R, in_features); up: (G, R, out_features), float16 or bfloat16,
    contiguous; scale: (G,) float32, or None for 1.  Adapters of a smaller
    rank are padded with zero rows."""

    down: Tensor
    up: Tensor
    scale: Tensor | None = None

    def __post_init__(self) -> None:
        if self.down.dim() != 3 or self.up.dim() != 3 or self.down.shape[:2] != self.up.shape[:2]:
            raise ValueError(f"down must be (G, R, in) and up (G, R, out), got {tuple(self.down.shape)} and "
                             f"{tuple(self.up.shape)}")
        if self.down.dtype != self.up.dtype:
            raise TypeError("down and up must share a dtype")
        if self.down.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"adapters must be float16 or bfloat16, got {self.down.dtype}")
        if not 1 <= self.down.shape[1] <= MAX_RANK or self.down.shape[2] < 1 or self.up.shape[2] < 1:
            raise ValueError(f"the rank must be 1 to {MAX_RANK} and the features positive")
        if not (self.down.is_contiguous() and self.up.is_contiguous()):
            raise ValueError("down and up must be contiguous")
        if self.scale is not None and (tuple(self.scale.shape) != (self.down.shape[0],)
                                       or self.scale.dtype != torch.float32 or not self.scale.is_contiguous()):
            raise ValueError(f"scale must be a contiguous ({self.down.shape[0]},) float32 tensor")
        for t in (self.up, self.scale):
            if t is not None and t.device != self.down.device:
                raise ValueError("down, up and scale must share a device")
        # What every call needs, read from the tensors once: (G, R, in, out) and the dtype's code.
        object.__setattr__(self, "_sizes", (*self.down.shape, self.up.shape[2]))
        object.__setattr__(self, "_code", _lib.kairo_dtype(self.down.dtype))

    @property
    def count(self) -> int:
        return self.down.shape[0]

    @property
    def rank(self) -> int:
        return self.down.shape[1]

    @property
    def in_features(self) -> int:
        return self.down.shape[2]

    @property
    def out_features(self) -> int:
        return self.up.shape[2]

    @property
    def dtype(self) -> torch.dtype:
        return self.down.dtype


@dataclass(frozen=True)
class AdapterPlan:
    """The tokens of a batch ordered by adapter (``adapter_plan``); opaque."""

    memory: Tensor
    num_tokens: int
    num_adapters: int


@functools.lru_cache(maxsize=4096)
def _plan_bytes(tokens: int, num_adapters: int) -> tuple[int, int]:
    size, ws = ctypes.c_size_t(0), ctypes.c_size_t(0)
    _lib.check(_lib.lib().kairo_adapter_plan_size(tokens, num_adapters, ctypes.byref(size), ctypes.byref(ws)),
               "adapter_plan")
    return size.value, max(ws.value, 256)


def adapter_plan(ids: Tensor, num_adapters: int) -> AdapterPlan:
    """Plan of a batch whose token t uses adapter ``ids[t]`` (int32 or int64,
    any shape, taken flat); an id outside [0, num_adapters), such as -1,
    means none.  Asynchronous, no read-back."""
    index = _lib.device_index("adapter_plan", ids)
    g = int(num_adapters)
    if g < 0:
        raise ValueError("num_adapters must be non-negative")
    flat = _flat_ids(ids, "adapter_plan")
    n = flat.numel()
    size, ws_size = _plan_bytes(n, g)
    mem = flat.new_empty(size, dtype=torch.uint8)
    ws = flat.new_empty(ws_size, dtype=torch.uint8)
    _lib.launch("adapter_plan", _lib.lib().kairo_adapter_plan_build, index, flat.data_ptr(), flat.element_size(), n, g,
                mem.data_ptr(), size, ws.data_ptr(), ws_size)
    return AdapterPlan(memory=mem, num_tokens=n, num_adapters=g)


def _check_batch(op: str, name: str, X, features: int, adapters: LowRankAdapters, plan: AdapterPlan) -> None:
    if X.shape != (plan.num_tokens, features):
        if len(X.shape) != 2 or X.shape[1] != features:
            raise ValueError(f"{op}: {name} must be (tokens, {features}), got {tuple(X.shape)}")
        raise ValueError(f"{op}: the plan is of {plan.num_tokens} tokens, {name} has {X.shape[0]}")
    if X.dtype != adapters.down.dtype:
        raise TypeError(f"{op}: {name} is {X.dtype}, the adapters are {adapters.down.dtype}")
    if plan.num_adapters != adapters._sizes[0]:
        raise ValueError(f"{op}: the plan is of {plan.num_adapters} adapters, not {adapters._sizes[0]}")


def _apply(op: str, index: int, X: Tensor, down: Tensor, up: Tensor, k: int, n: int, rank: int, code: int,
           scale: Tensor | None, plan: AdapterPlan, base: Tensor | None, out: Tensor | None,
           low: Tensor | None) -> None:
    if base is None:
        base_ptr, base_ld, base_dt = None, n, code
    else:
        base_ptr, base_ld, base_dt = base.data_ptr(), _ld(base), _lib.kairo_dtype(base.dtype)
    if out is None:
        out_ptr, out_ld, out_dt = None, n, code
    else:
        out_ptr, out_ld, out_dt = out.data_ptr(), _ld(out), _lib.kairo_dtype(out.dtype)
    _lib.launch(op, _lib.lib().kairo_low_rank_apply, index, X.data_ptr(), _ld(X), k, down.data_ptr(), up.data_ptr(), n,
                rank, code, None if scale is None else scale.data_ptr(), plan.memory.data_ptr(), plan.num_tokens,
                plan.num_adapters, base_ptr, base_ld, base_dt, out_ptr, out_ld, out_dt,
                None if low is None else low.data_ptr())


def _result(op: str, like: Tensor, shape: tuple[int, int], base: Tensor | None, out: Tensor | None,
            dtype: torch.dtype | None) -> tuple[Tensor | None, Tensor]:
    """The checked base (rows contiguous) and the tensor to write; ``like`` has the adapters' type and device."""
    own = like.dtype
    odt = dtype or (own if out is None else out.dtype)
    if odt != own and odt != torch.float32:
        raise TypeError(f"{op}: the output must be float32 or {own}, got {odt}")
    if base is not None:
        if base.shape != shape or base.get_device() != like.get_device():
            raise ValueError(f"{op}: base must be {shape} on {like.device}")
        if base.dtype != own and base.dtype != torch.float32:
            raise TypeError(f"{op}: base must be float32 or {own}, got {base.dtype}")
        base = _rows(base)
    if out is None:
        out = like.new_empty(shape) if odt == own else like.new_empty(shape, dtype=odt)
    elif out.shape != shape or out.dtype != odt or out.device != like.device or _rows(out) is not out:
        raise ValueError(f"{op}: out must be a row-major {shape} {odt} tensor on {like.device}")
    return base, out


def adapter_linear(X: Tensor, adapters: LowRankAdapters, plan: AdapterPlan, *, base: Tensor | None = None,
                   out_dtype: torch.dtype | None = None, out: Tensor | None = None,
                   return_low: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """``Y[t] = base[t] + scale[a] * (X[t] down[a]^T) up[a]`` for the adapter a of each token.

    X: (tokens, in_features) in the adapters' dtype; base: (tokens,
    out_features) in that dtype or float32, None for zero.  The sum is formed
    in fp32 and rounded once to ``out_dtype`` (default: the adapters').
    ``out`` may be ``base`` itself, and shares no memory with an input
    otherwise.  ``return_low=True`` also returns the
    (tokens, rank) float32 values ``scale[a] * X[t] down[a]^T`` that
    ``adapter_linear_backward`` takes.

    An infinity or a NaN in X, down, up or the scale makes the results that it
    enters non-finite (NaN where the sum would be infinite, too) and reaches
    no other token's."""
    op = "adapter_linear"
    _, rank, k, n = adapters._sizes
    index = _lib.device_index(op, X, adapters.down, plan.memory)
    _check_batch(op, "X", X, k, adapters, plan)
    if out is not None:
        in_place = base is not None and (base.data_ptr(), base.stride(), base.dtype) == (out.data_ptr(), out.stride(),
                                                                                         out.dtype)
        _lib.refuse_overlap(op, out, X, adapters.down, adapters.up, plan.memory,
                            *(t for t in (adapters.scale, None if in_place else base) if t is not None))
    base, out = _result(op, adapters.down, (plan.num_tokens, n), base, out, out_dtype)
    low = X.new_empty((plan.num_tokens, rank), dtype=torch.float32) if return_low else None
    _apply(op, index, _rows(X), adapters.down, adapters.up, k, n, rank, adapters._code, adapters.scale, plan, base, out,
           low)
    return (out, low) if return_low else out


def _wgrad(op: str, index: int, low: Tensor, Z: Tensor | QuantizedActivations, plan: AdapterPlan,
           dtype: torch.dtype) -> Tensor:
    rank, k = low.shape[1], Z.shape[1]
    grad = low.new_empty((plan.num_adapters, rank, k), dtype=dtype)
    tail = (k, _lib.kairo_dtype(Z.dtype), plan.memory.data_ptr(), plan.num_tokens, plan.num_adapters,
            grad.data_ptr(), _lib.kairo_dtype(dtype))
    if isinstance(Z, QuantizedActivations):
        _lib.launch(op, _lib.lib().kairo_low_rank_wgrad_q8, index, low.data_ptr(), rank, Z.codes.data_ptr(), Z._ldq,
                    Z.steps.data_ptr(), Z._lds, *tail)
    else:
        _lib.launch(op, _lib.lib().kairo_low_rank_wgrad, index, low.data_ptr(), rank, Z.data_ptr(), _ld(Z), *tail)
    return grad


def adapter_linear_backward(dY: Tensor, X: Tensor | QuantizedActivations | None, adapters: LowRankAdapters,
                            plan: AdapterPlan, *, low: Tensor | None = None, base_dx: Tensor | None = None,
                            need_dx: bool = True, need_dw: bool = True, dx_dtype: torch.dtype | None = None,
                            grad_dtype: torch.dtype | None = None
                            ) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """(dX, d_down, d_up) of ``adapter_linear``; the gradient by its base is dY.

    X may be given in 8 bits; with ``need_dw=False`` it is not read and may be
    None.  ``low``: what ``return_low`` gave (computed anew from X otherwise).
    ``base_dx``: the shared projection's part of dX, added in fp32 before the
    one rounding to ``dx_dtype`` (default: the adapters').  d_down and d_up are in ``grad_dtype`` (default: the
    adapters'), zero for an adapter without tokens.  Infinities and NaN: as in
    ``adapter_linear``."""
    op = "adapter_linear_backward"
    _, rank, k, n = adapters._sizes
    down, up, code = adapters.down, adapters.up, adapters._code
    tokens = plan.num_tokens
    kept = X if isinstance(X, QuantizedActivations) else None
    if need_dw and X is None:
        raise ValueError(f"{op}: the gradients of down and up need X")
    # X takes no part in dX
    index = _lib.device_index(op, dY, down, plan.memory, *((kept.codes if kept else X,) if need_dw else ()))
    _check_batch(op, "dY", dY, n, adapters, plan)
    gdt = grad_dtype or down.dtype
    if gdt != torch.float32 and gdt != down.dtype:
        raise TypeError(f"{op}: the gradients must be float32 or {down.dtype}, got {gdt}")
    if need_dw:
        _check_batch(op, "X", X, k, adapters, plan)
        if kept and low is None:
            raise ValueError(f"{op}: an X in 8 bits needs the low of the forward pass")
        if low is not None and (low.shape != (tokens, rank) or low.dtype != torch.float32
                                or low.get_device() != index):
            raise ValueError(f"{op}: low must be a ({tokens}, {rank}) float32 tensor")
    dX = None
    if need_dx:
        base_dx, dX = _result(op, down, (tokens, k), base_dx, None, dx_dtype)
    dY = _rows(dY)
    dlow = dY.new_empty((tokens, rank), dtype=torch.float32) if need_dw else None
    if need_dx or need_dw:
        _apply(op, index, dY, up, down, n, k, rank, code, adapters.scale, plan, base_dx if need_dx else None, dX, dlow)
    if not need_dw:
        return dX, None, None
    Z = kept or _rows(X)
    if low is None:
        low = torch.empty_like(dlow)
        _apply(op, index, Z, down, up, k, n, rank, code, adapters.scale, plan, None, None, low)
    low = low.contiguous()
    if kept:
        return dX, _wgrad(op, index, dlow, Z, plan, gdt), _wgrad(op, index, low, dY, plan, gdt)
    d_down = torch.empty_like(down) if gdt == down.dtype else down.new_empty(down.shape, dtype=gdt)
    d_up = torch.empty_like(up) if gdt == up.dtype else up.new_empty(up.shape, dtype=gdt)
    _lib.launch(op, _lib.lib().kairo_low_rank_wgrads, index, dlow.data_ptr(), low.data_ptr(), rank, Z.data_ptr(),
                _ld(Z), k, dY.data_ptr(), _ld(dY), n, code, plan.memory.data_ptr(), tokens, plan.num_adapters,
                d_down.data_ptr(), d_up.data_ptr(), _lib.kairo_dtype(gdt))
    return dX, d_down, d_up


def adapted_sparse_linear(X: Tensor, W: BlockSparseMatrix, adapters: LowRankAdapters, plan: AdapterPlan, *,
                          out_dtype: torch.dtype | None = None, config: KernelConfig | None = None,
                          return_low: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """``sparse_linear(X, W)`` plus each token's adapter: the projection's fp32
    result and the adapter's are added before the one rounding to
    ``out_dtype`` (default: X's)."""
    if tuple(W.shape) != (adapters.out_features, adapters.in_features):
        raise ValueError(f"W is {tuple(W.shape)}, the adapters are for "
                         f"({adapters.out_features}, {adapters.in_features})")
    odt = out_dtype or X.dtype
    base = sparse_linear(X, W, out_dtype=torch.float32, config=config)
    return adapter_linear(X, adapters, plan, base=base, out_dtype=odt,
                          out=base if odt == torch.float32 else None, return_low=return_low)


class _AdaptedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X: Tensor, blocks: Tensor, down: Tensor, up: Tensor, module: "AdaptedSparseLinear",
                plan: AdapterPlan) -> Tensor:
        layer = module.layer
        W = layer.weight_matrix(blocks)
        scale = module.scale
        Y, low = adapted_sparse_linear(X, W, module.adapters(down, up, scale), plan, return_low=True)
        need_x = any(ctx.needs_input_grad[1:4])
        kept: list[Tensor] = []
        ctx.kept_dtype = None
        if need_x and layer.checkpoint is not None:
            q = quantize_activations(X)
            kept, ctx.kept_dtype = list(q._parts()), q.dtype
        elif need_x:
            kept = [X]
        ctx.save_for_backward(blocks, down, up, scale, low, *kept)
        ctx.module, ctx.plan, ctx.need_x = module, plan, need_x
        return Y

    @staticmethod
    @once_differentiable
    def backward(ctx, dY: Tensor):
        blocks, down, up, scale, low, *kept = ctx.saved_tensors
        module: AdaptedSparseLinear = ctx.module
        layer = module.layer
        X = None
        if ctx.need_x:
            X = kept[0] if ctx.kept_dtype is None else QuantizedActivations._from_parts(*kept, layer.shape[1],
                                                                                         ctx.kept_dtype)
        W = layer.weight_matrix(blocks)
        dY = dY.contiguous()
        need_dx, need_blocks = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        need_dw = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        wt = transpose_values(W, layer.transposed()) if need_dx or need_blocks else None
        base_dx = sparse_linear(dY, wt.matrix, out_dtype=torch.float32) if need_dx else None
        dX = d_down = d_up = None
        if need_dx or need_dw:
            dX, d_down, d_up = adapter_linear_backward(dY, X, module.adapters(down, up, scale), ctx.plan, low=low,
                                                       base_dx=base_dx, need_dx=need_dx, need_dw=need_dw)
        d_blocks = sparse_linear_weight_grad(dY, X, W, wt, out_dtype=blocks.dtype) if need_blocks else None
        return dX, d_blocks, d_down, d_up, None, None


class AdaptedSparseLinear(torch.nn.Module):
    """A ``BlockSparseLinear`` with low-rank adapters: ``forward(X, plan)``.

    ``down`` (G, R, in_features) and ``up`` (G, R, out_features) are
    parameters; ``up`` starts at zero, so that a new adapter changes nothing.
    The layer's blocks train too unless frozen
    (``layer.blocks.requires_grad_(False)``).  A layer built with
    ``checkpoint="int8"`` keeps its input in 8 bits for all three
    gradients.

    A step's backward pass uses the ``scale`` of its forward pass.  Like the
    parameters it must not be written in between (autograd raises); to switch
    the adapters off for a pass, assign another tensor to ``scale``."""

    def __init__(self, layer: BlockSparseLinear, num_adapters: int, rank: int, *,
                 scale: float | Tensor = 1.0) -> None:
        super().__init__()
        out_features, in_features = layer.shape
        if num_adapters < 1 or not 1 <= rank <= MAX_RANK:
            raise ValueError(f"num_adapters must be positive and the rank 1 to {MAX_RANK}")
        dev, dt = layer.blocks.device, layer.blocks.dtype
        if dt not in (torch.float16, torch.bfloat16):
            raise TypeError(f"adapters must be float16 or bfloat16; the layer is {dt}")
        self.layer = layer
        self.down = torch.nn.Parameter((torch.randn(num_adapters, rank, in_features, device=dev)
                                        * in_features**-0.5).to(dt))
        self.up = torch.nn.Parameter(torch.zeros(num_adapters, rank, out_features, dtype=dt, device=dev))
        s = torch.as_tensor(scale, dtype=torch.float32, device=dev)
        self.register_buffer("scale", s.expand(num_adapters).clone())

    def _apply(self, fn, recurse: bool = True) -> "AdaptedSparseLinear":
        # .to(dtype), .half() and the like cast every floating buffer; scale stays in fp32
        kept = self.scale
        super()._apply(fn, recurse)
        if self.scale.dtype != torch.float32:
            self.scale = kept.to(self.scale.device)
        return self

    def adapters(self, down: Tensor | None = None, up: Tensor | None = None,
                 scale: Tensor | None = None) -> LowRankAdapters:
        return LowRankAdapters(down=(self.down if down is None else down).detach(),
                               up=(self.up if up is None else up).detach(),
                               scale=self.scale if scale is None else scale)

    def forward(self, X: Tensor, plan: AdapterPlan) -> Tensor:
        if not torch.is_grad_enabled():  # no backward pass: nothing to keep
            return adapted_sparse_linear(X, self.layer.weight_matrix(), self.adapters(), plan)
        return _AdaptedLinearFn.apply(X, self.layer.blocks, self.down, self.up, self, plan)
