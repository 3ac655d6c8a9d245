"""Scaled embedding lookup and its gradient by sorted tokens.

The plain implementation is in 64 bits.  A lookup is one fp32 product rounded
once: off by at most half a step of the output's type, and one of fp32 on the
way.  A gradient row is an fp32 sum of c products, whose rounding errors are
at most (c + 1) * 2^-24 of the sum of magnitudes, and one rounding to the
output's type.
"""

from __future__ import annotations

import pytest
import torch

from kairo_b200.ops import ScaledEmbedding, embedding_grad, embedding_lookup, sort_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _half(t):
    return torch.finfo(t).eps / 2


def _ids(n_rows, tokens, seed, skew=4.0, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(tokens, generator=g, dtype=torch.float64)
    return (n_rows * u**skew).long().clamp(max=max(n_rows - 1, 0)).to(dtype)


def _check_lookup(w, ids, scale, out):
    n = w.shape[0]
    flat = ids.reshape(-1).cpu().long()
    ok = (flat >= 0) & (flat < n)
    ref = torch.zeros(flat.numel(), w.shape[1], dtype=torch.float64)
    ref[ok] = w.double().cpu()[flat[ok]] * scale
    got = out.double().cpu().reshape(ref.shape)
    # half a step of the output, of fp32's product and of scale in fp32; below
    # the normal range the step is that of the subnormals
    tol = ref.abs() * (_half(out.dtype) * (1 + 1e-3) + 2 * 2.0**-24) + torch.finfo(out.dtype).smallest_normal * _half(
        out.dtype) * 2
    assert bool(((got - ref).abs() <= tol).all())


def _grad_ref(grad, ids, n_rows, scale):
    flat = ids.reshape(-1).cpu().long()
    g = grad.double().cpu().reshape(flat.numel(), -1)
    ok = (flat >= 0) & (flat < n_rows)
    ref = torch.zeros(n_rows, g.shape[1], dtype=torch.float64).index_add_(0, flat[ok], g[ok] * scale)
    mag = torch.zeros_like(ref).index_add_(0, flat[ok], g[ok].abs() * abs(scale))
    count = torch.zeros(n_rows, dtype=torch.float64).index_add_(0, flat[ok], torch.ones(int(ok.sum()),
                                                                                       dtype=torch.float64))
    return ref, mag, count


def _grad_tol(ref, mag, count, dtype):
    # fp32 sum of `count` terms, then the products with scale (and of scale
    # itself in fp32), then one rounding to dtype
    s = mag * (count[:, None] + 3) * 2.0**-24
    return s + (ref.abs() + s) * _half(dtype) * (1 + 1e-3) + torch.finfo(dtype).smallest_normal * _half(dtype) * 2


def _check_grad(grad, ids, n_rows, scale, out):
    ref, mag, count = _grad_ref(grad, ids, n_rows, scale)
    assert bool(((out.double().cpu() - ref).abs() <= _grad_tol(ref, mag, count, out.dtype)).all())


@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("ot", TYPES)
@pytest.mark.parametrize("case", [(1000, 64, 257), (37, 5, 12), (500, 4096, 3), (10, 1, 40), (300, 1037, 129)])
def test_lookup(wt, ot, case):
    n, d, t = case
    g = torch.Generator().manual_seed(n + d)
    w = torch.randn(n, d, generator=g).to(wt)
    ids = torch.randint(-2, n + 2, (t,), generator=g)
    for it in (torch.int32, torch.int64):
        out = embedding_lookup(w.to(DEV), ids.to(DEV, it), scale=8.5, out_dtype=ot)
        assert out.dtype == ot
        _check_lookup(w, ids, 8.5, out)


def test_lookup_shapes_strides_and_out():
    w = torch.randn(64, 96, device=DEV)
    ids = torch.randint(0, 64, (3, 7), device=DEV)
    assert embedding_lookup(w, ids).shape == (3, 7, 96)
    for view in (w[:, 8:72], w[:, 3:40], w[::2, :], w.t()):  # offset, unaligned, strided rows, transposed
        i = ids % view.shape[0]
        assert torch.equal(embedding_lookup(view, i), view[i])
    wide = torch.full((4, 7, 96), 3.0, device=DEV)
    out = embedding_lookup(w, ids, out=wide[:3])
    assert torch.equal(out, w[ids]) and bool((wide[3] == 3).all())
    assert embedding_lookup(w, ids[:0]).shape == (0, 7, 96)
    assert embedding_lookup(w, ids[0, 0]).shape == (96,)
    assert bool((embedding_lookup(w[:0], ids) == 0).all())  # a table of no rows: every id is out of range
    shifted = torch.empty(21 * 96 + 1, device=DEV)[1:].view(3, 7, 96)
    assert torch.equal(embedding_lookup(w, ids, out=shifted), w[ids])


@pytest.mark.parametrize("case", [
    # rows, tokens, skew: one pass, several tiles, three passes, one id, none in range
    (5, 1, 1.0), (200, 4096, 1.0), (255, 2049, 4.0), (256, 2047, 4.0), (70000, 5000, 4.0), (1 << 24, 9999, 1.0),
    (1, 3000, 1.0), (1000, 100001, 3.0),
])
@pytest.mark.parametrize("it", [torch.int32, torch.int64])
def test_sort_tokens(case, it):
    n, t, skew = case
    ids = _ids(n, t, seed=t, skew=skew, dtype=it)
    ids[::7] = -5
    ids[3::11] = n
    order = sort_tokens(ids.to(DEV), n)
    key = torch.where((ids < 0) | (ids >= n), n, ids.long())
    perm = torch.argsort(key, stable=True)
    assert torch.equal(order.perm.cpu().long(), perm)
    assert torch.equal(order.sorted_ids.cpu().long(), key[perm])


@pytest.mark.parametrize("gt,ot", [(a, b) for a in TYPES for b in TYPES])
@pytest.mark.parametrize("case", [
    # rows, dim, tokens, skew
    (1000, 64, 1, 1.0),
    (50, 5, 333, 1.0),
    (3000, 130, 4100, 4.0),     # several chunks of one id, a ragged column slice
    (4, 2048, 700, 1.0),        # every run crosses chunks
])
def test_grad(gt, ot, case):
    n, d, t, skew = case
    g = torch.Generator().manual_seed(t)
    grad = torch.randn(t, d, generator=g).to(gt)
    ids = _ids(n, t, seed=t, skew=skew)
    ids[5::9] = -1
    out = embedding_grad(grad.to(DEV), ids.to(DEV), n, scale=1.5, out_dtype=ot)
    assert out.dtype == ot
    _check_grad(grad, ids, n, 1.5, out)
    assert torch.equal(out, embedding_grad(grad.to(DEV), sort_tokens(ids.to(DEV, torch.int32), n), n, scale=1.5,
                                           out_dtype=ot))


@pytest.mark.parametrize("tokens", [255, 256, 257, 511, 512, 513, 4095, 4096, 4097, 65536, 65537])
@pytest.mark.parametrize("dim", [6, 67, 264])
def test_grad_at_the_list_lengths(tokens, dim):
    """Lists on both sides of every length at which the order is found in another way."""
    n = 90
    g = torch.Generator().manual_seed(tokens)
    grad = torch.randn(tokens, dim, generator=g).half()
    ids = _ids(n, tokens, seed=dim, skew=3.0)
    ids[2::13] = n
    order = sort_tokens(ids.to(DEV), n)
    key = torch.where(ids >= n, n, ids)
    assert torch.equal(order.perm.cpu().long(), torch.argsort(key, stable=True))
    out = embedding_grad(grad.to(DEV), ids.to(DEV), n, scale=0.5, out_dtype=torch.float32)
    _check_grad(grad, ids, n, 0.5, out)
    assert torch.equal(out, embedding_grad(grad.to(DEV), order, n, scale=0.5, out_dtype=torch.float32))


@pytest.mark.parametrize("tokens", [1, 31, 32, 33, 64, 65, 1000, 20000])
def test_grad_of_one_row(tokens):
    """All tokens share one id; the runs end before, at and behind chunk borders."""
    grad = torch.randn(tokens, 40, generator=torch.Generator().manual_seed(tokens))
    ids = torch.full((tokens,), 7)
    _check_grad(grad, ids, 9, 1.0, embedding_grad(grad.to(DEV), ids.to(DEV), 9))
    two = ids.clone()
    two[: tokens // 3] = 3
    _check_grad(grad, two, 9, 1.0, embedding_grad(grad.to(DEV), two.to(DEV), 9))


@pytest.mark.parametrize("ot", TYPES)
def test_grad_accumulates(ot):
    """Touched rows get base + sum (one rounding); the others keep their bits, NaN too."""
    n, d, t = 400, 72, 900
    g = torch.Generator().manual_seed(0)
    grad = torch.randn(t, d, generator=g)
    ids = _ids(n, t, seed=1)
    base = torch.randn(n, d, generator=g).to(ot)
    count = torch.bincount(ids, minlength=n)
    base[count == 0] = float("nan")
    wide = torch.zeros(n, d + 8, dtype=ot, device=DEV)
    out = wide[:, :d]
    out.copy_(base)
    got = embedding_grad(grad.to(DEV), ids.to(DEV), n, scale=0.25, out=out, accumulate=True)
    assert got is out and bool((wide[:, d:] == 0).all())
    touched = count > 0
    assert bool(out[~touched.to(DEV)].isnan().all())
    ref, mag, cnt = _grad_ref(grad, ids, n, 0.25)
    ref = ref[touched] + base[touched].double()
    mag = mag[touched] + base[touched].double().abs()
    tol = _grad_tol(ref, mag, cnt[touched], ot)
    assert bool(((out[touched.to(DEV)].double().cpu() - ref).abs() <= tol).all())


def test_grad_edges():
    g = torch.randn(6, 12, device=DEV)
    none = torch.full((6,), -1, device=DEV)
    assert bool((embedding_grad(g, none, 5) == 0).all())                         # every token is padding
    assert bool((embedding_grad(g[:0], none[:0], 5) == 0).all())                 # no tokens
    assert embedding_grad(g, none, 0).shape == (0, 12)                           # no rows
    ids = torch.tensor([[0, 1, 2], [2, 1, 4]], device=DEV)
    ref = torch.zeros(5, 12, device=DEV).index_add_(0, ids.flatten(), g)
    assert torch.allclose(embedding_grad(g.view(2, 3, 12), ids, 5), ref, rtol=0, atol=1e-6)
    strided = torch.randn(6, 40, device=DEV)[:, 3:15]                            # unaligned rows
    ref = torch.zeros(5, 12, device=DEV).index_add_(0, ids.flatten(), strided)
    assert torch.allclose(embedding_grad(strided.unflatten(0, (2, 3)), ids, 5), ref, rtol=0, atol=1e-6)
    one = torch.randn(1, 12, device=DEV).expand(6, 12)                           # a broadcast gradient
    ref = torch.zeros(5, 12, device=DEV).index_add_(0, ids.flatten(), one)
    assert torch.allclose(embedding_grad(one, ids.flatten(), 5), ref, rtol=0, atol=1e-6)
    inf = torch.zeros(6, 12, device=DEV)
    inf[2, 3], inf[4, 5] = float("inf"), float("nan")
    got = embedding_grad(inf, ids.flatten(), 5)
    assert got[2, 3].isinf() and got[1, 5].isnan() and int(got.isfinite().sum()) == 58


def test_grad_row_offsets_pass_32_bits():
    """A table of more than 2^31 elements: the last rows are read and written where they belong."""
    n, d = 1_100_000, 2048
    w = torch.zeros(n, d, dtype=torch.float16, device=DEV)
    ids = torch.tensor([n - 1, 5, n - 2, n - 1], device=DEV)
    w[n - 1], w[n - 2], w[5] = 3.0, 2.0, 1.0
    assert embedding_lookup(w, ids)[:, 7].tolist() == [3.0, 1.0, 2.0, 3.0]
    del w
    g = torch.ones(4, d, dtype=torch.float16, device=DEV)
    out = embedding_grad(g, ids, n)
    assert out[n - 1].unique().tolist() == [2.0] and out[5].unique().tolist() == [1.0]
    assert int(torch.count_nonzero(out.sum(1, dtype=torch.float32))) == 3


def test_module_gradient_and_differences():
    m = ScaledEmbedding(50, 16, scale=4.0, device=DEV)
    ids = torch.randint(0, 50, (8, 3), device=DEV)
    c = torch.randn(8, 3, 16, device=DEV)
    (m(ids) * c).sum().backward()
    ref = torch.zeros(50, 16, dtype=torch.float64).index_add_(0, ids.flatten().cpu(),
                                                             4.0 * c.double().cpu().view(-1, 16))
    assert bool(((m.weight.grad.double().cpu() - ref).abs() <= 26 * 2.0**-24 * 4.0 * c.abs().max().item() * 2).all())
    # the loss is linear in the table, so a difference of any size gives the derivative; fp64 sums of fp32 outputs
    i, j, h = int(ids[0, 0]), 3, 0.5
    with torch.no_grad():
        up = (m(ids).double() * c).sum()
        m.weight[i, j] += h
        diff = ((m(ids).double() * c).sum() - up) / h
    # each of the (at most 24) outputs of row i moved by 4 h with an error of a few 2^-24 of its value
    tol = 24 * c.abs().max().item() * 4 * (m.weight[i, j].abs().item() + 2 * h) * 4 * 2.0**-24 / h
    assert abs(diff.item() - m.weight.grad[i, j].item()) <= tol + 1e-6
    half = ScaledEmbedding(50, 16, out_dtype=torch.bfloat16, device=DEV)
    out = half(ids)
    assert out.dtype == torch.bfloat16
    out.float().sum().backward()
    assert half.weight.grad.dtype == torch.float32


def test_streams_and_graph():
    n, d, t = 5000, 256, 3000
    w = torch.randn(n, d, device=DEV)
    ids = _ids(n, t, seed=3).to(DEV)
    grad = torch.randn(t, d, device=DEV)
    ref_f, ref_g = embedding_lookup(w, ids, scale=2.0), embedding_grad(grad, ids, n, scale=2.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f, g = embedding_lookup(w, ids, scale=2.0), embedding_grad(grad, ids, n, scale=2.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(f, ref_f) and torch.equal(g, ref_g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        f, g = embedding_lookup(w, ids, scale=2.0), embedding_grad(grad, ids, n, scale=2.0)
    new = _ids(n, t, seed=4).to(DEV)
    ids.copy_(new)
    grad.normal_()
    for _ in range(2):
        f.fill_(float("nan"))
        g.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(f, embedding_lookup(w, new, scale=2.0))
        assert torch.equal(g, embedding_grad(grad, new, n, scale=2.0))


def test_out_must_not_share_memory():
    w = torch.randn(20, 16, device=DEV)
    ids = torch.arange(4, device=DEV)
    with pytest.raises(ValueError, match="share memory"):
        embedding_lookup(w, ids, out=w[2:6])
    with pytest.raises(ValueError, match="share memory"):
        embedding_grad(w[:4], ids, 20, out=w)
    embedding_lookup(w, ids, out=torch.empty(4, 16, device=DEV))
    with pytest.raises(TypeError):
        embedding_lookup(w, ids.float())
    with pytest.raises(ValueError):
        embedding_grad(w[:3], ids, 20)
    with pytest.raises(ValueError):
        embedding_grad(w[:4], ids, 20, accumulate=True)
    with pytest.raises(ValueError):
        embedding_grad(w[:4], sort_tokens(ids, 19), 20)


def test_second_derivative_is_refused():
    m = ScaledEmbedding(10, 8, device=DEV)
    out = m(torch.arange(4, device=DEV))
    (g,) = torch.autograd.grad(out.square().sum(), m.weight, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("tokens", [400, 3000, 70000])
def test_two_calls_at_once(tokens):
    """Gradients of two batches on two streams, started together, with no work between them to order them."""
    n, d = 700, 64
    grads = [torch.randn(tokens, d, device=DEV) for _ in range(2)]
    ids = [_ids(n, tokens, seed=i, skew=3.0).to(DEV) for i in range(2)]
    ref = [embedding_grad(g, i, n) for g, i in zip(grads, ids)]
    _check_grad(grads[0], ids[0], n, 1.0, ref[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    out = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[k].append(embedding_grad(grads[k], ids[k], n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref[k]) for k in range(2) for o in out[k])
