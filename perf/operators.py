"""Cases and plain forms of the operators around the block-sparse linear layer.

Three groups of operators, each in both directions where it is trained:

* embedding: the scaled lookup of token rows and its gradient, summed per row
  over tokens sorted by id;
* checkpoints: activations kept in 8 bits for the backward pass, read back
  whole or used directly by the weight gradient of the block-sparse linear
  layer;
* adapters: low-rank adapters of many requests in one batch, added to a
  shared projection's output, for single tokens, prompts and training.

``run`` computes them in elementary torch operations in 32 bits (``own``
false) or through kairo_b200 (``own`` true).
"""

import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_GROUP = 64      # columns that share one scale of an 8-bit checkpoint
_SKEW = 4.0      # token id = N * u**4: the most frequent token takes N**-0.25 of the text


def listed():
    return [
        # One decoding step of 64 sequences: latency of one launch.
        {"name": "lookup_decode", "op": "lookup", "rows": 131072, "dim": 4096, "tokens": 64, "dtype": "bf16",
         "out": "bf16", "scale": 64.0},
        # A recommender's fp32 table (the embedding benchmark's size) read for a bf16 model.
        {"name": "lookup_batch_f32_table", "op": "lookup", "rows": 1000000, "dim": 128, "tokens": 65536,
         "dtype": "f32", "out": "bf16", "scale": 11.3125},
        # Small fp32 table and batch (the reference's embedding benchmark).
        {"name": "embed_grad_small", "op": "embed_grad", "rows": 10000, "dim": 64, "tokens": 256, "dtype": "f32",
         "out": "f32", "scale": 1.0},
        # A training batch of skewed text over a large vocabulary.
        {"name": "embed_grad_train", "op": "embed_grad", "rows": 131072, "dim": 2048, "tokens": 32768,
         "dtype": "bf16", "out": "bf16", "scale": 45.25},
        # A ragged activation kept and read back whole (a consumer without a fused form).
        {"name": "checkpoint_ragged", "op": "checkpoint", "tokens": 333, "cols": 1000, "dtype": "f16"},
        # Weight gradient of a mid-sized sparse layer, fp32 gradients, from a checkpoint made in the forward pass.
        {"name": "checkpoint_grad_mid", "op": "checkpoint_grad", "tokens": 2048, "rows": 4096, "cols": 4096,
         "keep": 0.2, "dtype": "f16", "out": "f32"},
        # The same at the linear-layer workload's size (8192 x 32768, 20 % of the blocks, batch 8192).
        {"name": "checkpoint_grad_linear", "op": "checkpoint_grad", "tokens": 8192, "rows": 8192, "cols": 32768,
         "keep": 0.2, "dtype": "bf16", "out": "bf16"},
        # One request decodes: latency.
        {"name": "adapters_single_token", "op": "adapters", "tokens": 1, "cols": 4096, "rows": 4096, "rank": 16,
         "adapters": 8, "order": "mixed", "dtype": "bf16", "out": "bf16"},
        # A serving batch: every token its own request, 64 adapters loaded, some requests without one.
        {"name": "adapters_decode_mixed", "op": "adapters", "tokens": 96, "cols": 8192, "rows": 8192, "rank": 16,
         "adapters": 64, "order": "mixed", "dtype": "bf16", "out": "bf16"},
        # Prompts of several requests packed into one batch at the linear-layer workload's width.
        {"name": "adapters_prompts", "op": "adapters", "tokens": 8192, "cols": 32768, "rows": 8192, "rank": 16,
         "adapters": 12, "order": "packed", "dtype": "bf16", "out": "bf16"},
        # Training with an odd batch and a rank that is no power of two, fp16, fp32 adapter gradients.
        {"name": "adapters_train_odd", "op": "adapters_train", "tokens": 777, "cols": 1000, "rows": 520, "rank": 12,
         "adapters": 5, "order": "packed", "dtype": "f16", "out": "f32"},
        # Fine-tuning several adapters at once beside a frozen projection.
        {"name": "adapters_train", "op": "adapters_train", "tokens": 8192, "cols": 8192, "rows": 8192, "rank": 32,
         "adapters": 4, "order": "packed", "dtype": "bf16", "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "embed_grad", "checkpoint", "checkpoint_grad", "adapters", "adapters",
                     "adapters_train"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op in ("lookup", "embed_grad"):
        dtype = rng.choice(["bf16", "f16", "f32"])
        dim = 8 * _log(rng, 8, 512) if rng.random() < 0.6 else _log(rng, 50, 3000)
        return {"op": op, "rows": _log(rng, 1000, 100000), "dim": dim, "tokens": _log(rng, 1, 40000), "dtype": dtype,
                "out": rng.choice(["f32", dtype]), "scale": rng.choice([1.0, math.sqrt(dim)])}
    if op == "checkpoint":
        return {"op": op, "tokens": _log(rng, 1, 9000), "cols": _log(rng, 60, 9000),
                "dtype": rng.choice(["bf16", "f16", "f32"])}
    if op == "checkpoint_grad":
        return {"op": op, "tokens": _log(rng, 100, 8000), "rows": 64 * _log(rng, 4, 100), "cols": 64 * _log(rng, 4, 200),
                "keep": rng.choice([0.1, 0.2, 0.5]), "dtype": dtype, "out": rng.choice(["f32", dtype])}
    odd = rng.random() < 0.3
    cols, rows = (_log(rng, 100, 9000), _log(rng, 100, 9000)) if odd else (64 * _log(rng, 8, 200), 64 * _log(rng, 8, 128))
    case = {"op": op, "cols": cols, "rows": rows, "rank": rng.choice([4, 8, 12, 16, 32, 64]),
            "adapters": _log(rng, 1, 48), "order": rng.choice(["mixed", "packed"]), "dtype": dtype}
    case["tokens"] = _log(rng, 1, 8000) if op == "adapters" else _log(rng, 16, 8000)
    case["out"] = rng.choice(["f32", dtype]) if op == "adapters_train" else dtype
    return case


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(std)


def _activations(g, n, k, dtype):
    """Hidden states as a layer meets them: unit scale, a few columns ten times larger, a few dead tokens."""
    x = _randn(g, n, k, dtype=dtype)
    loud = torch.rand(k, generator=g, device="cuda") < 0.002
    x.mul_(torch.where(loud, 10.0, 1.0).to(dtype))
    dead = torch.rand(n, generator=g, device="cuda") < 0.002
    return x.masked_fill_(dead[:, None], 0.0)


def _token_ids(g, rows, tokens, skew):
    u = torch.rand(tokens, generator=g, device="cuda", dtype=torch.float64)
    return (rows * u**skew).long().clamp_(max=rows - 1)


def _request_ids(g, case):
    """The adapter of every token: packed prompts of uneven lengths, or one token per request; -1 has none."""
    t, n = case["tokens"], case["adapters"]
    if case["order"] == "mixed":
        ids = torch.randint(0, n, (t,), generator=g, device="cuda")
        return torch.where(torch.rand(t, generator=g, device="cuda") < 0.06, -1, ids) if t > 8 else ids
    cuts = torch.sort(torch.rand(max(n - 1, 0), generator=g, device="cuda")).values * t
    ids = torch.searchsorted(cuts, torch.arange(t, device="cuda") + 0.5)
    if n > 3:
        ids = torch.where(ids == 2, -1, ids)  # one request goes without an adapter, so one adapter has no token
    return ids


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    dt = _DT[case["dtype"]]
    s = {"case": case}
    if op == "lookup":
        s["weight"] = _randn(g, case["rows"], case["dim"], std=0.02, dtype=dt)
        s["ids"] = _token_ids(g, case["rows"], case["tokens"], 1.0)
    elif op == "embed_grad":
        s["grad"] = _randn(g, case["tokens"], case["dim"], std=0.01, dtype=dt)
        s["ids"] = _token_ids(g, case["rows"], case["tokens"], _SKEW)
    elif op == "checkpoint":
        s["x"] = _activations(g, case["tokens"], case["cols"], dt)
    elif op == "checkpoint_grad":
        s["x"] = _activations(g, case["tokens"], case["cols"], dt)
        s["dy"] = _randn(g, case["tokens"], case["rows"], std=0.01, dtype=dt)
        nbr, nbc = case["rows"] // 64, case["cols"] // 64
        keep = max(1, int(nbr * nbc * case["keep"]))
        pos = torch.sort(torch.randperm(nbr * nbc, generator=g, device="cuda")[:keep]).values
        s["rows"], s["cols"] = pos // nbc, pos % nbc
        if own:
            from kairo_b200.ops import bsr_from_tiles, bsr_transpose

            blocks = torch.zeros(keep, 64, 64, dtype=dt, device="cuda")
            s["w"] = bsr_from_tiles(blocks, s["rows"].int(), s["cols"].int(), (case["rows"], case["cols"]))
            s["wt"] = bsr_transpose(s["w"])
    else:
        n, r = case["adapters"], case["rank"]
        s["x"] = _activations(g, case["tokens"], case["cols"], dt)
        s["down"] = _randn(g, n, r, case["cols"], std=case["cols"] ** -0.5, dtype=dt)
        s["up"] = _randn(g, n, r, case["rows"], std=0.3 * r**-0.5, dtype=dt)
        s["scale"] = 0.5 + 1.5 * torch.rand(n, generator=g, device="cuda")
        s["ids"] = _request_ids(g, case)
        s["base"] = _randn(g, case["tokens"], case["rows"], dtype=dt)
        if op == "adapters_train":
            s["dy"] = _randn(g, case["tokens"], case["rows"], std=0.01, dtype=dt)
            s["base_dx"] = _randn(g, case["tokens"], case["cols"], std=0.01, dtype=dt)
        if own:
            from kairo_b200.ops import LowRankAdapters, adapter_plan

            s["adapters"] = LowRankAdapters(down=s["down"], up=s["up"], scale=s["scale"])
            s["plan"] = adapter_plan(s["ids"], n)
    return s


# ---------------------------------------------------------------- plain forms


def _plain_checkpoint(x):
    """Codes round(x * 127 / amax) of every 64 columns of a row, read back as code * (amax / 127) in x's type.
    The product that decides the rounding is exact in 64 bits."""
    n, k = x.shape
    pad = -k % _GROUP
    xf = torch.nn.functional.pad(x.float(), (0, pad)).view(n, -1, _GROUP)
    amax = xf.abs().amax(dim=2, keepdim=True)
    live = amax >= 2.0**-100
    inv = torch.where(live, 127.0 / amax, 0.0)
    codes = (xf.double() * inv.double()).round().clamp(-127, 127).float()
    back = codes * torch.where(live, amax / 127.0, 0.0)
    return back.view(n, -1)[:, :k].to(x.dtype)


def _plain_low(s):
    """Rows of every adapter beside one another, (tokens, adapters * rank), zero for the adapters of other tokens."""
    n, r, k = s["down"].shape
    mine = s["ids"][:, None] == torch.arange(n, device="cuda")[None, :]
    mask = (mine.float() * s["scale"][None, :]).repeat_interleave(r, dim=1)
    return s["x"].float() @ s["down"].float().view(n * r, k).t(), mask


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "lookup":
        return (s["weight"][s["ids"]].float() * case["scale"]).to(_DT[case["out"]])
    if op == "embed_grad":
        acc = torch.zeros(case["rows"], case["dim"], device="cuda")
        acc.index_add_(0, s["ids"], s["grad"].float())
        return (acc * case["scale"]).to(_DT[case["out"]])
    if op == "checkpoint":
        return _plain_checkpoint(s["x"])
    if op == "checkpoint_grad":
        xh = _plain_checkpoint(s["x"]).float()
        dense = s["dy"].float().t() @ xh
        nbr, nbc = case["rows"] // 64, case["cols"] // 64
        return dense.view(nbr, 64, nbc, 64)[s["rows"], :, s["cols"], :].to(_DT[case["out"]])
    n, r, k = s["down"].shape
    low, mask = _plain_low(s)
    up = s["up"].float().view(n * r, -1)
    y = (s["base"].float() + (low * mask) @ up).to(s["base"].dtype)
    if op == "adapters":
        return y
    dlow = (s["dy"].float() @ up.t()) * mask
    dx = (s["base_dx"].float() + dlow @ s["down"].float().view(n * r, k)).to(s["x"].dtype)
    odt = _DT[case["out"]]
    ddown = (dlow.t() @ s["x"].float()).view(n, r, k).to(odt)
    dup = ((low * mask).t() @ s["dy"].float()).view(n, r, -1).to(odt)
    return {"y": y, "dx": dx, "ddown": ddown, "dup": dup}


# ---------------------------------------------------------------- the framework's calls


def _own(s):
    from kairo_b200 import ops

    case = s["case"]
    op = case["op"]
    if op == "lookup":
        return ops.embedding_lookup(s["weight"], s["ids"], scale=case["scale"], out_dtype=_DT[case["out"]])
    if op == "embed_grad":
        return ops.embedding_grad(s["grad"], s["ids"], case["rows"], scale=case["scale"], out_dtype=_DT[case["out"]])
    if op == "checkpoint":
        return ops.dequantize_activations(ops.quantize_activations(s["x"]))
    if op == "checkpoint_grad":
        kept = ops.quantize_activations(s["x"])
        return ops.sparse_linear_weight_grad(s["dy"], kept, s["w"], s["wt"], out_dtype=_DT[case["out"]])
    if op == "adapters":
        return ops.adapter_linear(s["x"], s["adapters"], s["plan"], base=s["base"])
    y, low = ops.adapter_linear(s["x"], s["adapters"], s["plan"], base=s["base"], return_low=True)
    dx, ddown, dup = ops.adapter_linear_backward(s["dy"], s["x"], s["adapters"], s["plan"], low=low,
                                                 base_dx=s["base_dx"], grad_dtype=_DT[case["out"]])
    return {"y": y, "dx": dx, "ddown": ddown, "dup": dup}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- the definition, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        return torch.index_select(s["weight"], 0, s["ids"]).double() * case["scale"]
    if op == "embed_grad":
        order = torch.argsort(s["ids"], stable=True)
        ids, counts = torch.unique_consecutive(s["ids"][order], return_counts=True)
        ends = torch.cumsum(counts, 0).tolist()
        g = s["grad"].double()[order] * case["scale"]
        out = torch.zeros(case["rows"], case["dim"], dtype=torch.float64, device="cuda")
        single = counts == 1
        first = torch.cumsum(counts, 0) - counts
        out[ids[single]] = g[first[single]]
        for j in torch.nonzero(~single).flatten().tolist():
            out[ids[j]] = g[ends[j] - int(counts[j]):ends[j]].sum(0)
        return out
    if op in ("checkpoint", "checkpoint_grad"):
        x = s["x"].double()
        back = torch.empty_like(x)
        for c in range(0, case["cols"], _GROUP):
            part = x[:, c:c + _GROUP]
            amax = part.abs().amax(1, keepdim=True).float()
            inv = (127.0 / amax).double()
            step = (amax / 127.0).double()
            value = torch.round(part * inv) * step
            back[:, c:c + _GROUP] = torch.where(amax >= 2.0**-100, value, torch.zeros_like(value))
        if op == "checkpoint":
            return back
        back = back.float().to(s["x"].dtype).double()  # a checkpoint reads back in the activation's own type
        dy = s["dy"].double()
        out = torch.empty(s["rows"].numel(), 64, 64, dtype=torch.float64, device="cuda")
        for j in torch.unique(s["cols"]).tolist():
            at = torch.nonzero(s["cols"] == j).flatten()
            g = dy.t() @ back[:, 64 * j:64 * j + 64]
            out[at] = g.view(-1, 64, 64)[s["rows"][at]]
        return out
    x, down, up, scale = s["x"].double(), s["down"].double(), s["up"].double(), s["scale"].double()
    y = s["base"].double()
    train = op == "adapters_train"
    if train:
        dy, dx = s["dy"].double(), s["base_dx"].double()
        ddown, dup = torch.zeros_like(down), torch.zeros_like(up)
    for a in range(case["adapters"]):
        at = torch.nonzero(s["ids"] == a).flatten()
        low = x[at] @ down[a].t()
        y[at] += scale[a] * (low @ up[a])
        if train:
            dlow = scale[a] * (dy[at] @ up[a].t())
            dx[at] += dlow @ down[a]
            ddown[a] = dlow.t() @ x[at]
            dup[a] = scale[a] * (low.t() @ dy[at])
    return {"y": y, "dx": dx, "ddown": ddown, "dup": dup} if train else y


# ---------------------------------------------------------------- what a pass cannot do without


def _distinct(rows, tokens, skew):
    """Expected number of different ids among `tokens` draws of rows * u**skew."""
    edge = (np.arange(rows + 1) / rows) ** (1.0 / skew)
    return float(-np.expm1(tokens * np.log1p(-np.minimum(np.diff(edge), 1 - 1e-12))).sum())


def work(case):
    op = case["op"]
    t = case["tokens"]
    e = _SIZE[case["dtype"]]
    if op == "lookup":
        d = case["dim"]
        return {"bytes": t * 8 + _distinct(case["rows"], t, 1.0) * d * e + t * d * _SIZE[case["out"]], "flops": t * d}
    if op == "embed_grad":
        d = case["dim"]
        return {"bytes": t * 8 + t * d * e + case["rows"] * d * _SIZE[case["out"]], "flops": t * d}
    if op == "checkpoint":
        return {"bytes": 2 * t * case["cols"] * e, "flops": 4 * t * case["cols"]}
    if op == "checkpoint_grad":
        m, k = case["rows"], case["cols"]
        blocks = max(1, int((m // 64) * (k // 64) * case["keep"]))
        return {"bytes": t * (m + k) * e + blocks * 4096 * _SIZE[case["out"]], "flops": 2 * blocks * 4096 * t}
    m, k, r, n = case["rows"], case["cols"], case["rank"], case["adapters"]
    used = n * (1 - (1 - 1 / n) ** t) if case["order"] == "mixed" else n
    nbytes = t * (k + 2 * m) * e + used * r * (k + m) * e
    flops = 2 * t * r * (k + m)
    if op == "adapters_train":
        nbytes += t * (m + 2 * k) * e + n * r * (k + m) * _SIZE[case["out"]]
        flops *= 3
    return {"bytes": nbytes, "flops": flops}
