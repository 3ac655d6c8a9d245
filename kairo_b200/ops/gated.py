"""Gated projection of a feed-forward block with block-sparse weights (CUDA only).

    G = X Wg^T      U = X Wu^T      H = act(G) * U

Both products, the activation and the product of the two are one kernel: G and
U are not in memory, neither in the forward pass nor for the backward pass,
which forms them again from X.

* ``gated_weights(gate, up)`` -- two block-sparse weights of one shape, laid out
  side by side once.
* ``sparse_gated_linear`` -- H, for single tokens and prompts alike.
* ``sparse_gated_linear_backward`` -- the gradients by X and by both weights'
  blocks.
* ``SparseGatedLinear`` -- both as a module with autograd;
  ``SparseFeedForward`` -- the whole block, ``down(act(gate(X)) * up(X))``.

The reference has no counterpart.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, field, replace

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from kairo_b200 import _lib
from kairo_b200.ops.backward import BlockSparseLinear, bsr_transpose
from kairo_b200.ops.spmm import KernelConfig, _bsr_desc
from kairo_b200.ops.token_embedding import _ld, _rows
from kairo_b200.types import BlockSparseMatrix

_ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}
_ANY_TOKENS = 8  # up to here X may have any alignment


@dataclass(frozen=True)
class GatedWeights:
    """Gate and up weights of one gated projection (``gated_weights``).

    blocks: (gate_blocks + up_blocks, b, b), the gate's in its BSR order, then
    the up weight's; the gradients come in this order (``split``).  The other
    tensors describe the patterns: ent_ptr / entries, the block-columns of every
    block-row with the two weights' blocks, and ``stacked``, the pattern of the
    (2 ceil(out / b) b, in) matrix whose block-rows 2i and 2i + 1 are block-row
    i of gate and of up."""

    blocks: Tensor
    gate_blocks: int
    shape: tuple[int, int]
    block: int
    ent_ptr: Tensor
    entries: Tensor
    row_ptr: Tensor   # of the stacked matrix
    col_idx: Tensor   # its block-columns, in its order
    blk_idx: Tensor   # stored block of each of its blocks
    stored_col: Tensor  # block-column of every stored block
    _structure: dict = field(default_factory=dict, repr=False, compare=False)

    def __post_init__(self) -> None:
        if self.blocks.dim() != 3 or self.blocks.shape[1:] != (self.block, self.block) or not self.blocks.is_contiguous():
            raise ValueError(f"blocks must be a contiguous (n, {self.block}, {self.block}) tensor")
        if self.blocks.shape[0] != self.stored_col.numel():
            raise ValueError(f"the patterns have {self.stored_col.numel()} blocks, got {self.blocks.shape[0]}")
        if self.blocks.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"gated weights must be float16 or bfloat16, got {self.blocks.dtype}")
        if self.blocks.device != self.entries.device:
            raise ValueError("blocks must be on the patterns' device")
        if self.blocks.data_ptr() % 16:
            raise ValueError("blocks must be 16-byte aligned")
        d = _lib.KairoGated()
        d.rows, d.cols = self.shape
        d.nentries, d.nblocks = self.entries.shape[0], self.blocks.shape[0]
        d.ent_ptr, d.entries, d.blocks = self.ent_ptr.data_ptr(), self.entries.data_ptr(), self.blocks.data_ptr()
        d.block, d.dtype = self.block, _lib.kairo_dtype(self.blocks.dtype)
        object.__setattr__(self, "_desc", d)

    @property
    def dtype(self) -> torch.dtype:
        return self.blocks.dtype

    @property
    def device(self) -> torch.device:
        return self.blocks.device

    # copied and pickled as tensors and numbers; the descriptor names this object's memory, and the structure is made again
    def __getstate__(self) -> dict:
        return {k: v for k, v in self.__dict__.items() if k not in ("_desc", "_structure")}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state, _structure={})
        self.__post_init__()

    def with_blocks(self, blocks: Tensor) -> "GatedWeights":
        """The same patterns with other values."""
        return replace(self, blocks=blocks)

    def split(self, blocks: Tensor) -> tuple[Tensor, Tensor]:
        """The gate's and the up weight's part of a tensor in ``blocks``' order."""
        return blocks[:self.gate_blocks], blocks[self.gate_blocks:]

    def matrices(self) -> tuple[BlockSparseMatrix, BlockSparseMatrix]:
        """Gate and up as BlockSparseMatrix views of ``blocks``."""
        out = []
        rp = self.row_ptr.to(torch.int64)
        for part, blocks in enumerate(self.split(self.blocks)):
            counts = rp[part + 1::2] - rp[part::2][:rp[part + 1::2].numel()]
            row_ptr = torch.zeros(counts.numel() + 1, dtype=torch.int32, device=self.device)
            row_ptr[1:] = torch.cumsum(counts, 0)
            cols = self.split(self.stored_col)[part].contiguous()
            out.append(BlockSparseMatrix(row_ptr=row_ptr, col_idx=cols, blocks=blocks, shape=self.shape,
                                         block_size=(self.block, self.block)))
        return out[0], out[1]

    def stacked(self) -> BlockSparseMatrix:
        """The stacked matrix (see above) over ``blocks``."""
        rows = (self.row_ptr.numel() - 1) * self.block
        return BlockSparseMatrix(row_ptr=self.row_ptr, col_idx=self.col_idx, blocks=self.blocks,
                                 shape=(rows, self.shape[1]), block_size=(self.block, self.block),
                                 blk_idx=self.blk_idx)

    def _backward_structure(self) -> "_Structure":
        """What the backward products need beside the values; made once per pattern."""
        made = self._structure.get("backward")
        if made is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("sparse_gated_linear_backward: the first backward pass of a pattern makes its "
                                   "transposed structure and synchronises; run one before capturing")
            made = self._structure["backward"] = _Structure(self)
        return made


class _Structure:
    """The stacked matrix transposed (structure only), descriptors and workspace sizes of the backward products.
    It serves values of both types: a descriptor's type and blocks are those of the call (``_with_blocks``)."""

    def __init__(self, w: GatedWeights) -> None:
        a = w.stacked()
        try:
            t = bsr_transpose(a, check=True)
        except _lib.KairoDeviceError as e:
            if e.code & 0xFF != _lib.DEVERR_ROW_TOO_LONG:
                raise
            raise ValueError("sparse_gated_linear_backward: a block-column keeps more than 16384 blocks of gate and up "
                             "together, more than the transposed structure is sorted for") from e
        self.kept = (t.matrix.row_ptr, t.matrix.col_idx, t.perm, w.row_ptr, w.col_idx, w.blk_idx, w.stored_col)
        # positions of the transposed structure name stored blocks, so that the weight gradient lands in the blocks' own order
        self.perm_stored = w.blk_idx[t.perm.long()] if a.nnzb else t.perm
        # the next call to find the structure may be on another stream
        stream = torch.cuda.current_stream(w.device)
        stream.synchronize()
        self.streams = {stream.cuda_stream}
        self.desc = _bsr_desc(a)
        self.desc_t = _bsr_desc(t.matrix)
        self.desc_w = _bsr_desc(BlockSparseMatrix(row_ptr=w.row_ptr, col_idx=w.stored_col, blocks=w.blocks,
                                                  shape=a.shape, block_size=a.block_size))
        self.spmm_bytes: dict[tuple[int, torch.dtype], int] = {}  # by tokens and type
        self.rows_t, self.longest_t = t.matrix.nbr, t.matrix.max_row_blocks
        nbytes = ctypes.c_size_t(0)
        _lib.check(_lib.lib().kairo_bsr_sddmm_workspace_size(ctypes.byref(self.desc_w), ctypes.byref(nbytes)), "sddmm")
        self.sddmm_bytes = max(nbytes.value, 256)

    def used_on_current_stream(self, index: int) -> None:
        """Before a call's launches: memory that only this object names must outlive them.  Work of another stream
        than the one it was made on is recorded with the allocator; a captured graph may replay at any time, whatever
        has become of the weights, so what it reads is kept for good."""
        raw = torch._C._cuda_getCurrentRawStream(index)
        if raw not in self.streams:
            stream = torch.cuda.current_stream(index)
            for t in (*self.kept, self.perm_stored):
                t.record_stream(stream)
            self.streams.add(raw)
        if torch.cuda.is_current_stream_capturing() and self not in _CAPTURED:
            _CAPTURED.append(self)

    def config(self, nnzb: int, tokens: int) -> _lib.KairoSpmmConfig:
        """Schedule of dP times the stacked weight.  Whole block-rows per CTA (bands of one) beat the row-split
        schedule, the library's own choice for few block-rows, from about 128 tokens on: it cuts nearly every
        row into partial tiles (6000 tokens, 512 -> 512: 25 us against 1469; 1000 tokens, 8192 -> 8192 at 20 %:
        107 against 126; 128 tokens, 16384 -> 4096: 62 against 32).  Tiles of 128 tokens where those of 256 do
        not fill the 148 SMs (777 tokens, 520 -> 1000: 19.5 us against 23.6).  A few rows far longer than the
        others would leave most SMs idle: split there."""
        if tokens <= 128 or self.longest_t > 8 * nnzb / max(self.rows_t, 1) + 8:
            return _AUTO
        return _BANDS_128 if self.rows_t * -(-tokens // 256) < 148 else _BANDS_256


_CAPTURED: list[_Structure] = []
_AUTO = KernelConfig().to_c()
_BANDS_128 = KernelConfig(schedule="bands", band_rows=1, n_tile=128).to_c()
_BANDS_256 = KernelConfig(schedule="bands", band_rows=1, n_tile=256).to_c()


def _with_blocks(desc: _lib.KairoBsr, blocks: Tensor) -> _lib.KairoBsr:
    d = _lib.KairoBsr.from_buffer_copy(desc)
    d.blocks, d.dtype = blocks.data_ptr(), _lib.kairo_dtype(blocks.dtype)
    return d


def _in_order(a: BlockSparseMatrix) -> Tensor:
    return a.blocks[:a.nnzb] if a.blk_idx is None else a.blocks[a.blk_idx.long()]


def gated_weights(gate: BlockSparseMatrix, up: BlockSparseMatrix) -> GatedWeights:
    """Lays out two block-sparse weights (out_features x in_features) of one
    shape, block size (16, 32 or 64, square) and type (float16 or bfloat16) for
    ``sparse_gated_linear``.  Their patterns may differ; neither may hold a
    block twice.  The blocks are copied.  Synchronises."""
    if not (gate.blocks.is_cuda and up.blocks.is_cuda):
        raise RuntimeError("kairo_b200.gated_weights runs on CUDA tensors only; this package has no CPU implementation")
    if gate.shape != up.shape or gate.block_size != up.block_size:
        raise ValueError(f"gate is {gate.shape} in blocks of {gate.block_size}, up is {up.shape} in blocks of "
                         f"{up.block_size}")
    if gate.dtype != up.dtype or gate.device != up.device:
        raise TypeError("gate and up must share a dtype and a device")
    if gate.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"gated weights must be float16 or bfloat16, got {gate.dtype}")
    b = gate.block_size[0]
    if gate.block_size[1] != b or b not in (16, 32, 64):
        raise ValueError(f"blocks must be 16 x 16, 32 x 32 or 64 x 64, got {gate.block_size}")
    dev, nbr, nbc = gate.device, gate.nbr, gate.nbc
    rows, keys = [], []
    for a in (gate, up):
        counts = (a.row_ptr[1:] - a.row_ptr[:-1]).long()
        if a.nnzb and (int(counts.min()) < 0 or int(a.row_ptr[0]) != 0 or int(a.row_ptr[-1]) != a.nnzb
                       or int(a.col_idx.min()) < 0 or int(a.col_idx.max()) >= nbc):
            raise ValueError("a weight's row_ptr or col_idx is malformed")
        r = torch.repeat_interleave(torch.arange(nbr, device=dev), counts, output_size=a.nnzb)
        rows.append(r)
        keys.append(r * nbc + a.col_idx.long())
    n_gate, n_up = gate.nnzb, up.nnzb
    merged, at = torch.unique(torch.cat(keys), return_inverse=True)
    entries = torch.full((merged.numel(), 4), -1, dtype=torch.int32, device=dev)
    entries[:, 0] = merged % max(nbc, 1)
    entries[:, 3] = 0
    for part, (lo, n) in enumerate(((0, n_gate), (n_gate, n_up))):
        mine = at[lo:lo + n]
        if torch.unique(mine).numel() != n:
            raise ValueError("a weight holds the same block twice")
        entries[mine, 1 + part] = torch.arange(lo, lo + n, dtype=torch.int32, device=dev)
    ent_ptr = torch.searchsorted(merged, torch.arange(nbr + 1, device=dev) * nbc).to(torch.int32)
    # the stacked matrix: row i of gate, row i of up, row i + 1 of gate, ...
    gp, up_ptr = gate.row_ptr.long(), up.row_ptr.long()
    row_ptr = torch.empty(2 * nbr + 1, dtype=torch.int64, device=dev)
    row_ptr[0::2] = gp + up_ptr
    row_ptr[1::2] = gp[1:] + up_ptr[:-1]
    place = torch.cat([torch.arange(n_gate, device=dev) + up_ptr[rows[0]],
                       torch.arange(n_up, device=dev) + gp[rows[1] + 1]])
    stored_col = torch.cat([gate.col_idx, up.col_idx])
    blk_idx = torch.empty(n_gate + n_up, dtype=torch.int32, device=dev)
    blk_idx[place] = torch.arange(n_gate + n_up, dtype=torch.int32, device=dev)
    col_idx = stored_col[blk_idx.long()]
    return GatedWeights(blocks=torch.cat([_in_order(gate), _in_order(up)]), gate_blocks=n_gate, shape=tuple(gate.shape),
                        block=b, ent_ptr=ent_ptr, entries=entries, row_ptr=row_ptr.to(torch.int32), col_idx=col_idx,
                        blk_idx=blk_idx, stored_col=stored_col)


def _input(op: str, X: Tensor, weights: GatedWeights, activation: str) -> tuple[Tensor, int]:
    """X as rows that the kernels read (a copy where they must be 16-byte aligned and are not), activation code."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{op}: activation must be one of {', '.join(_ACTIVATIONS)}, got {activation!r}")
    k = weights.shape[1]
    if X.dim() != 2 or X.shape[1] != k:
        raise ValueError(f"{op}: Inner dimensions must match: X is {tuple(X.shape)}, the weights are {weights.shape}")
    if X.dtype != weights.dtype:
        raise TypeError(f"{op}: X is {X.dtype}, the weights are {weights.dtype}")
    return _rows(X), _ACTIVATIONS[activation]


def _aligned(X: Tensor) -> Tensor:
    n, k = X.shape
    if X.data_ptr() % 16 == 0 and (n <= 1 or X.stride(0) % 8 == 0):
        return X
    out = X.new_empty((n, -(-k // 8) * 8))[:, :k]
    return out.copy_(X)


def sparse_gated_linear(X: Tensor, weights: GatedWeights, *, activation: str = "silu", out: Tensor | None = None,
                        check: bool = False) -> Tensor:
    """``act(X Wg^T) * (X Wu^T)``: (tokens, out_features) in X's type, from fp32 sums, rounded once.

    X: (tokens, in_features) in the weights' type.  activation: "silu", "gelu"
    (by erf), "gelu_tanh" or "relu".  ``out``: a row-major tensor to write to,
    sharing no memory with an input.

    A value of X that is not finite makes those results non-finite whose row
    keeps a block of gate or up in its column, and no others.  ``check=True``
    synchronises and raises KairoDeviceError where a kernel met a malformed
    entry or a wait ran out; without it ``pending_device_error`` tells."""
    op = "sparse_gated_linear"
    index = _lib.device_index(op, X, weights.blocks)
    x, act = _input(op, X, weights, activation)
    n, m = x.shape[0], weights.shape[0]
    if n > _ANY_TOKENS:
        x = _aligned(x)
    if out is None:
        out = x.new_empty((n, m))
    elif out.shape != (n, m) or out.dtype != x.dtype or out.device != x.device or _rows(out) is not out:
        raise ValueError(f"{op}: out must be a row-major ({n}, {m}) {x.dtype} tensor on {x.device}")
    else:
        _lib.refuse_overlap(op, out, X, weights.blocks)
    err = _lib.error_word(index)
    if check:
        _lib.take_pending_error(err, op)
    _lib.launch(op, _lib.lib().kairo_gated_linear, index, ctypes.byref(weights._desc), x.data_ptr(),
                max(_ld(x), weights.shape[1]), n, act, out.data_ptr(), _ld(out), err.data_ptr())
    if check:
        _lib.raise_on_device_error(err)
    return out


def sparse_gated_linear_backward(dH: Tensor, X: Tensor, weights: GatedWeights, *, activation: str = "silu",
                                 need_dx: bool = True, need_dw: bool = True, dw_dtype: torch.dtype | None = None,
                                 check: bool = False) -> tuple[Tensor | None, Tensor | None]:
    """(dX, d_blocks) of ``sparse_gated_linear``: dX in X's type; d_blocks in
    ``dw_dtype`` (default: the weights'; or float32), in the order of
    ``weights.blocks`` (``weights.split`` gives the two weights' parts).
    Either may be left out (None).

    dG and dU are rounded to the weights' type, as operands of both products.
    A block-column may keep 16384 blocks, gate and up together (ValueError).
    ``check=True`` synchronises and raises KairoDeviceError where one of the
    kernels met a malformed structure or a wait ran out; without it
    ``pending_device_error`` tells."""
    op = "sparse_gated_linear_backward"
    index = _lib.device_index(op, dH, X, weights.blocks)
    x, act = _input(op, X, weights, activation)
    n, (m, k) = x.shape[0], weights.shape
    if dH.shape != (n, m):
        raise ValueError(f"{op}: dH must be ({n}, {m}), got {tuple(dH.shape)}")
    if dH.dtype != x.dtype:
        raise TypeError(f"{op}: dH is {dH.dtype}, X is {x.dtype}")
    dwt = dw_dtype or weights.dtype
    if dwt not in (torch.float32, weights.dtype):
        raise TypeError(f"{op}: dw_dtype must be float32 or {weights.dtype}, got {dwt}")
    if not (need_dx or need_dw):
        return None, None
    x, dh = _aligned(x), _rows(dH)
    nbr = weights.ent_ptr.numel() - 1
    dp = x.new_empty((n, 2 * nbr * weights.block))
    err = _lib.error_word(index)
    if check:
        _lib.take_pending_error(err, op)
    _lib.launch(op, _lib.lib().kairo_gated_linear_grad, index, ctypes.byref(weights._desc), x.data_ptr(),
                max(_ld(x), k), n, act, dh.data_ptr(), max(_ld(dh), m), dp.data_ptr(), dp.shape[1], err.data_ptr())
    if check:
        _lib.raise_on_device_error(err)
    nnzb, b = weights.blocks.shape[0], weights.block
    dX = d_blocks = None
    if nnzb == 0 or n == 0:
        dX = x.new_zeros((n, k)) if need_dx else None
        return dX, weights.blocks.new_zeros(weights.blocks.shape, dtype=dwt) if need_dw else None
    lib = _lib.lib()
    st = weights._backward_structure()
    st.used_on_current_stream(index)
    if need_dx:
        # the transposed weight's values are of this call alone: the structure serves calls on several streams
        blocks_t = weights.blocks.new_empty((nnzb, b, b))
        # its workspace is an error word and nothing else
        _lib.launch(op, lib.kairo_bsr_transpose_values, index, ctypes.byref(_with_blocks(st.desc, weights.blocks)),
                    st.kept[2].data_ptr(), blocks_t.data_ptr(), err.data_ptr(), 256)
        desc_t, cfg = _with_blocks(st.desc_t, blocks_t), st.config(nnzb, n)
        dX = x.new_empty((n, k))
        size = st.spmm_bytes.get((n, x.dtype))
        if size is None:
            nbytes = ctypes.c_size_t(0)
            with torch.cuda.device(index):
                _lib.check(lib.kairo_bsr_spmm_workspace_size(ctypes.byref(desc_t), _lib.LAYOUT_LINEAR, n,
                                                             ctypes.byref(cfg), ctypes.byref(nbytes)), op)
            size = nbytes.value
            if len(st.spmm_bytes) < 4096:
                st.spmm_bytes[n, x.dtype] = size
        ws = _lib.workspace(size, x.device)
        if check:
            _lib.take_pending_error(ws, op)
        _lib.launch(op, lib.kairo_bsr_spmm, index, ctypes.byref(desc_t), dp.data_ptr(), dp.shape[1],
                    _lib.LAYOUT_LINEAR, n, dX.data_ptr(), k, _lib.kairo_dtype(x.dtype), ctypes.byref(cfg),
                    ws.data_ptr(), ws.numel())
        _lib.report_captured(op, index, ws)
        if check:
            _lib.raise_on_device_error(ws)
    if need_dw:
        d_blocks = weights.blocks.new_empty((nnzb, b, b), dtype=dwt)
        ws = x.new_empty(st.sddmm_bytes, dtype=torch.uint8)
        _lib.launch(op, lib.kairo_bsr_sddmm_word, index, ctypes.byref(_with_blocks(st.desc_w, weights.blocks)),
                    st.kept[0].data_ptr(), st.kept[1].data_ptr(), st.perm_stored.data_ptr(), dp.data_ptr(), dp.shape[1],
                    x.data_ptr(), max(_ld(x), k), n, d_blocks.data_ptr(), _lib.kairo_dtype(dwt), ws.data_ptr(),
                    ws.numel(), err.data_ptr())
    if check:
        _lib.raise_on_device_error(err)
    return dX, d_blocks


_PATTERN = ("ent_ptr", "entries", "row_ptr", "col_idx", "blk_idx", "stored_col")
# of a layer's buffers: the buffers, their versions, the kept structure, copies for backward passes by stream
_NOTHING: tuple = ((), (), {}, {})


class _GatedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X: Tensor, blocks: Tensor, module: "SparseGatedLinear") -> Tensor:
        w = module.weights(blocks)
        H = sparse_gated_linear(X, w, activation=module.activation)
        # all that the backward pass needs is this call's: the module may have changed by then
        ctx.save_for_backward(X, blocks)
        ctx.activation = module.activation
        ctx.weights = {"gate_blocks": w.gate_blocks, "shape": w.shape, "block": w.block, "_structure": w._structure,
                       **dict(zip(_PATTERN, module._pattern_of_call(X.get_device())))}
        return H

    @staticmethod
    @once_differentiable
    def backward(ctx, dH: Tensor):
        X, blocks = ctx.saved_tensors
        w = GatedWeights(blocks=blocks.detach(), **ctx.weights)
        dX, dW = sparse_gated_linear_backward(dH, X, w, activation=ctx.activation, need_dx=ctx.needs_input_grad[0],
                                              need_dw=ctx.needs_input_grad[1])
        return dX, dW, None


class SparseGatedLinear(torch.nn.Module):
    """``act(X Wg^T) * (X Wu^T)`` with block-sparse weights of fixed patterns.

    The parameter is ``blocks``: the gate's blocks in BSR order, then the up
    weight's (``gate_blocks`` of them are the gate's)."""

    def __init__(self, gate: BlockSparseMatrix, up: BlockSparseMatrix, *, activation: str = "silu") -> None:
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}, got {activation!r}")
        w = gated_weights(gate, up)
        self.activation = activation
        self.shape = w.shape
        self.gate_blocks = w.gate_blocks
        self.block = w.block
        self.blocks = torch.nn.Parameter(w.blocks.detach())
        for name in _PATTERN:
            self.register_buffer(name, getattr(w, name))
        self._made: tuple = _NOTHING

    def __getstate__(self) -> dict:
        # a copy makes its own structure: this one's descriptors name this layer's memory
        return {**self.__dict__, "_made": _NOTHING}

    def _load_from_state_dict(self, *args, **kw) -> None:
        super()._load_from_state_dict(*args, **kw)
        # patterns of as many blocks in all may give the gate another number of them
        if not self.row_ptr.is_meta:
            self.gate_blocks = int((self.row_ptr[1::2] - self.row_ptr[0:-1:2]).sum())

    def weights(self, blocks: Tensor | None = None) -> GatedWeights:
        b = (self.blocks if blocks is None else blocks).detach()
        parts = tuple(getattr(self, name) for name in _PATTERN)
        # the patterns' transposed structure is kept until a buffer is replaced or written (load_state_dict);
        # writes of inference tensors are not counted, so nothing is kept for them
        structure: dict = {}
        if not any(p.is_inference() for p in parts):
            versions = tuple(p._version for p in parts)
            if self._made[1] != versions or any(p is not q for p, q in zip(self._made[0], parts)):
                self._made = (parts, versions, structure, {})
            structure = self._made[2]
        return GatedWeights(blocks=b, gate_blocks=self.gate_blocks, shape=self.shape, block=self.block,
                            _structure=structure, **dict(zip(_PATTERN, parts)))

    def _pattern_of_call(self, index: int) -> list[Tensor]:
        """The patterns that ``weights`` has just given, for the backward pass.  Copies, as the buffers may be written
        before it (by a state dict, or a broadcast before the model's next forward pass): one set for each writing of
        the buffers and stream, on which autograd runs the backward pass as well.  In a capture the buffers
        themselves, which the graph's forward pass reads."""
        parts, _, _, copies = self._made
        if torch.cuda.is_current_stream_capturing():
            return [getattr(self, name) for name in _PATTERN]
        if not parts:  # inference tensors: nothing is kept
            return [getattr(self, name).clone() for name in _PATTERN]
        raw = torch._C._cuda_getCurrentRawStream(index)
        if raw not in copies:
            copies[raw] = [p.clone() for p in parts]
        return copies[raw]

    def forward(self, X: Tensor) -> Tensor:
        if not torch.is_grad_enabled():
            return sparse_gated_linear(X, self.weights(), activation=self.activation)
        return _GatedFn.apply(X, self.blocks, self)


class SparseFeedForward(torch.nn.Module):
    """The feed-forward block ``down(act(gate(X)) * up(X))`` of a ``SparseGatedLinear`` and a ``BlockSparseLinear``."""

    def __init__(self, gate: BlockSparseMatrix, up: BlockSparseMatrix, down: BlockSparseMatrix, *,
                 activation: str = "silu", checkpoint: str | None = None) -> None:
        super().__init__()
        if down.shape[1] != gate.shape[0]:
            raise ValueError(f"down is {down.shape}, gate and up have {gate.shape[0]} outputs")
        self.gated = SparseGatedLinear(gate, up, activation=activation)
        self.down = BlockSparseLinear(down, checkpoint=checkpoint)

    def forward(self, X: Tensor) -> Tensor:
        return self.down(self.gated(X))
