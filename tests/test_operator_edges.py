"""Corners of the operators around the linear layer that need no device: what a
call hands to the library, and what modules keep, with the library faked
where a call would launch."""

from __future__ import annotations

import contextlib

import pytest
import torch

from kairo_b200 import _lib
from kairo_b200.ops import (
    AdaptedSparseLinear,
    AdapterPlan,
    BlockSparseLinear,
    LowRankAdapters,
    QuantizedActivations,
    TokenOrder,
    adapter_linear,
    adapter_linear_backward,
    adapters,
    backward,
)
from kairo_b200.types import BlockSparseMatrix


def _bsr(dtype=torch.float32, m=64, k=64):
    nbr, nbc = -(-m // 64), -(-k // 64)
    return BlockSparseMatrix(row_ptr=torch.arange(nbr + 1, dtype=torch.int32) * nbc,
                             col_idx=torch.arange(nbc, dtype=torch.int32).repeat(nbr),
                             blocks=torch.zeros(nbr * nbc, 64, 64, dtype=dtype), shape=(m, k), block_size=(64, 64))


class _FakeLib:
    """Records the arguments of every call; each succeeds and does nothing."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] = args
            return _lib.SUCCESS

        return call


@pytest.fixture
def fake(monkeypatch):
    lib = _FakeLib()
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(_lib, "stream_handle", lambda dev: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(backward, "_require_cuda", lambda *t, op: None)
    return lib


@pytest.mark.parametrize("dy", [
    torch.ones(64).expand(300, 64),            # a broadcast gradient: every row the same memory
    torch.ones(300 * 8 + 64).as_strided((300, 64), (8, 1)),  # rows that overlap
    torch.ones(300, 80)[:, :64],
    torch.ones(64, 300).t(),
    torch.ones(1, 64),
])
def test_weight_grad_reads_inside_dy(fake, dy):
    """The rows that the library is told to read lie inside the gradient's memory."""
    n = dy.shape[0]
    seen = {}
    contiguous = torch.Tensor.contiguous

    def note(t):
        out = contiguous(t)
        seen[out.data_ptr()] = out
        return out

    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(torch.Tensor, "contiguous", note)
        q = QuantizedActivations(codes=torch.zeros(n, 64, dtype=torch.int8), steps=torch.zeros(1, n),
                                 dtype=torch.float32)
        wt = backward.TransposedBsr(matrix=_bsr(), perm=torch.zeros(1, dtype=torch.int32))
        backward.sparse_linear_weight_grad(dy, q, _bsr(), wt)
    ptr, lddy = fake.calls["kairo_bsr_sddmm_q8"][4:6]
    used = seen.get(ptr, dy)
    room = used.untyped_storage().nbytes() // 4 - used.storage_offset()
    assert ptr == used.data_ptr() and lddy >= 64 and (n - 1) * lddy + 64 <= room


def test_backward_without_x(monkeypatch):
    """dX alone takes no X; the other gradients say that they need one."""
    down, up = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 4, 32, dtype=torch.bfloat16)
    a = LowRankAdapters(down=down, up=up)
    plan = AdapterPlan(memory=torch.zeros(256, dtype=torch.uint8), num_tokens=3, num_adapters=2)
    dy = torch.zeros(3, 32, dtype=torch.bfloat16)
    seen = []
    monkeypatch.setattr(_lib, "device_index", lambda op, *t: seen.append([x.get_device() for x in t]) or -1)
    monkeypatch.setattr(_lib, "launch", lambda *args: None)
    dx, dd, du = adapter_linear_backward(dy, None, a, plan, need_dw=False)
    assert dx.shape == (3, 64) and dd is None and du is None and len(seen) == 1
    with pytest.raises(ValueError, match="need X"):
        adapter_linear_backward(dy, None, a, plan)


def test_scale_stays_in_fp32():
    """Casting a model leaves the adapters' scale in the type and with the values that the kernels take."""
    scale = torch.tensor([1.0, 1 / 3, 1e-30])
    for cast in (lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.bfloat16(),
                 lambda m: torch.nn.Sequential(m).to(torch.float16)[0], lambda m: m.double().bfloat16(), lambda m: m.to("cpu")):
        layer = AdaptedSparseLinear(BlockSparseLinear(_bsr(torch.bfloat16)), 3, 4, scale=scale)
        layer = cast(layer)
        assert layer.scale.dtype == torch.float32 and torch.equal(layer.scale, scale)
        assert "scale" in dict(layer.named_buffers()) and layer.adapters().count == 3
    layer = AdaptedSparseLinear(BlockSparseLinear(_bsr(torch.bfloat16)), 3, 4).to("meta")
    assert layer.scale.device.type == "meta"


@pytest.mark.parametrize("n,k", [(5, 100), (1, 100), (3, 64), (1, 16), (4, 1), (0, 100)])
@pytest.mark.parametrize("pitch", [0, 48])
def test_checkpoint_parts_survive_copies(n, k, pitch):
    """The parts that a backward pass keeps can be cloned or moved, and read back with rows of 16-byte pitch."""
    ldq = -(-k // 16) * 16 + pitch
    codes = torch.randint(-127, 128, (n, ldq), dtype=torch.int8)[:, :k]
    q = QuantizedActivations(codes=codes, steps=torch.rand(-(-k // 64), n), dtype=torch.bfloat16)
    for copy in (lambda t: t, lambda t: t.clone(), lambda t: torch.empty(t.size(), dtype=t.dtype).copy_(t)):
        back = QuantizedActivations._from_parts(*(copy(t) for t in q._parts()), k, q.dtype)
        assert torch.equal(back.codes, codes) and torch.equal(back.steps, q.steps) and back.dtype == q.dtype
        assert back._ldq % 16 == 0


@pytest.mark.parametrize("n,k", [(1, 100), (1, 1), (3, 100)])
def test_codes_without_their_padding_are_refused(n, k):
    """The kernels read whole 16-byte vectors: the last row's must lie inside the tensor's memory."""
    ldq = -(-k // 16) * 16
    steps = torch.ones(-(-k // 64), n)
    full = torch.zeros(n * ldq, dtype=torch.int8)
    QuantizedActivations(codes=full.view(n, ldq)[:, :k], steps=steps, dtype=torch.float32)
    short = full[: (n - 1) * ldq + k].clone().as_strided((n, k), (ldq, 1))
    with pytest.raises(ValueError, match="padded to 16"):
        QuantizedActivations(codes=short, steps=steps, dtype=torch.float32)
    if n == 1:  # the copy of a single row
        with pytest.raises(ValueError, match="padded to 16"):
            QuantizedActivations(codes=torch.zeros(1, k, dtype=torch.int8), steps=steps, dtype=torch.float32)


def test_token_order_refusals():
    """A token order is passed on as two pointers and a length: its parts must fit them."""
    ids, perm = torch.tensor([0, 2, 5], dtype=torch.int32), torch.tensor([1, 0, 2], dtype=torch.int32)
    assert TokenOrder(sorted_ids=ids, perm=perm, num_embeddings=5).num_embeddings == 5
    for bad in ({"perm": perm.long()}, {"sorted_ids": ids.long()}, {"sorted_ids": ids[:2]}, {"perm": perm[:2]},
                {"perm": perm.view(1, 3)}, {"perm": torch.zeros(6, dtype=torch.int32)[::2]},
                {"sorted_ids": torch.zeros(3, 2, dtype=torch.int32)[:, 0]}, {"sorted_ids": ids.to("meta")}):
        with pytest.raises(ValueError):
            TokenOrder(**{"sorted_ids": ids, "perm": perm, "num_embeddings": 5, **bad})


def test_overlap():
    """Refused: memory that is shared.  Columns of one wider matrix, side by side, share none."""
    buf = torch.zeros(8, 20)
    out = buf[:, 4:10]

    def refused(t, o=out):
        try:
            _lib.refuse_overlap("op", o, t)
        except ValueError:
            return True
        return False

    mine = {x.data_ptr() for x in (out[i, j] for i in range(8) for j in range(6))}
    for c0 in range(20):
        for c1 in range(c0 + 1, 21):
            for r0, r1 in ((0, 8), (2, 7), (3, 5)):
                t = buf[r0:r1, c0:c1]
                theirs = {x.data_ptr() for x in (t[i, j] for i in range(r1 - r0) for j in range(c1 - c0))}
                assert refused(t) == bool(mine & theirs), (c0, c1, r0, r1)
    half = buf.view(torch.float16)  # rows of the same bytes in another type
    assert not refused(half[:, :8]) and refused(half[:, :9]) and not refused(half[:, 20:]) and refused(half[:, 19:])
    # where the pitches differ, any meeting of the spans counts
    assert refused(buf.view(-1)[:40]) and refused(buf[::2, 12:]) and refused(buf.t()) and not refused(buf.clone())
    assert not refused(buf[:, 4:4]) and refused(out) and refused(buf[0, 4].expand(3, 6))
    assert not refused(buf.view(-1)[:4]) and not refused(buf.view(-1)[150:])


def test_out_is_compared_with_every_input(monkeypatch):
    """adapter_linear's result may not lie over its scale or its plan either."""
    down, up = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 4, 32, dtype=torch.bfloat16)
    monkeypatch.setattr(_lib, "device_index", lambda op, *t: -1)
    monkeypatch.setattr(_lib, "launch", lambda *args: None)
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    out = torch.zeros(3, 32)
    plain = LowRankAdapters(down=down, up=up)
    plan = AdapterPlan(memory=torch.zeros(256, dtype=torch.uint8), num_tokens=3, num_adapters=2)
    assert adapter_linear(x, plain, plan, out=out) is out
    with pytest.raises(ValueError, match="share memory"):
        adapter_linear(x, LowRankAdapters(down=down, up=up, scale=out.view(-1)[5:7]), plan, out=out)
    over = AdapterPlan(memory=out.view(-1).view(torch.uint8)[:256], num_tokens=3, num_adapters=2)
    with pytest.raises(ValueError, match="share memory"):
        adapter_linear(x, plain, over, out=out)


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_nothing_is_kept_without_a_backward_pass(monkeypatch, mode):
    """Without gradients a layer with 8-bit checkpoints quantises nothing."""
    calls = []
    x = torch.zeros(3, 64)
    for module in (adapters, backward):
        monkeypatch.setattr(module, "quantize_activations", lambda t: calls.append(t) or QuantizedActivations(
            codes=torch.zeros(3, 64, dtype=torch.int8), steps=torch.zeros(1, 3), dtype=t.dtype))
    monkeypatch.setattr(backward, "sparse_linear", lambda X, W, **kw: torch.ones(3, 64))
    monkeypatch.setattr(adapters, "adapted_sparse_linear", lambda X, W, a, plan, return_low=False: (
        (torch.ones(3, 64), torch.zeros(3, 4)) if return_low else torch.ones(3, 64)))
    plain = BlockSparseLinear(_bsr(), checkpoint="int8")
    adapted = AdaptedSparseLinear(BlockSparseLinear(_bsr(torch.bfloat16), checkpoint="int8"), 2, 4)
    with mode():
        for y in (plain(x), adapted(x, None)):
            assert y.shape == (3, 64) and not y.requires_grad
    assert not calls
    assert plain(x).requires_grad and adapted(x, None).requires_grad and len(calls) == 2
