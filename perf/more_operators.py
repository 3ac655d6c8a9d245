"""Cases and plain forms of the operators at both ends of a block-sparse model's layer stack.

Two groups of operators, in both directions where they are trained:

* loss: softmax cross entropy of hidden states against a whole vocabulary
  table (the embedding's own, when tied), without keeping the logits: token
  scores when serving, the loss and the gradients by hidden states and table
  when training;
* gated: the feed-forward block's gated projection act(X Wg^T) * (X Wu^T) with
  block-sparse Wg and Wu: single tokens, prompts, and the gradients by X and
  both weights.

``run`` computes them in elementary torch operations in 32 bits (``own``
false) or through kairo_b200 (``own`` true).
"""

import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16}
_SKEW = 4.0  # token id = V * u**4: the most frequent token takes V**-0.25 of the text


def listed():
    return [
        # Training step at the reference's embedding benchmark's size: latency of the launches.
        {"name": "loss_train_small", "op": "loss_train", "tokens": 256, "vocab": 10000, "dim": 64, "dtype": "bf16",
         "scale": 1.0, "reduction": "mean"},
        # Log-probability of one token over a large vocabulary while decoding.
        {"name": "loss_score_one", "op": "loss", "tokens": 1, "vocab": 131072, "dim": 4096, "dtype": "bf16",
         "scale": 1.0, "reduction": "none"},
        # The same for a decoding step of 64 sequences, fp16, with the logits scaled.
        {"name": "loss_score_batch", "op": "loss", "tokens": 64, "vocab": 131072, "dim": 4096, "dtype": "f16",
         "scale": 0.5, "reduction": "none"},
        # Perplexity of a validation batch; a ragged vocabulary and width.
        {"name": "loss_eval", "op": "loss", "tokens": 4000, "vocab": 50021, "dim": 1000, "dtype": "bf16",
         "scale": 1.0, "reduction": "mean"},
        # Fine-tuning with a weight per token; odd sizes throughout, rows of the table that are not 16-byte aligned.
        {"name": "loss_train_odd", "op": "loss_train", "tokens": 333, "vocab": 32003, "dim": 1001, "dtype": "f16",
         "scale": 1.0, "reduction": "none"},
        # A training batch over a large vocabulary (the table of the embedding's gradient case).
        {"name": "loss_train", "op": "loss_train", "tokens": 8192, "vocab": 131072, "dim": 2048, "dtype": "bf16",
         "scale": 1.0, "reduction": "mean"},
        # One request decodes through the widest layer, gate and up pruned apart.
        {"name": "gated_one_token", "op": "gated", "tokens": 1, "cols": 8192, "rows": 32768, "block": 64, "keep": 0.2,
         "pattern": "own", "act": "silu", "dtype": "bf16"},
        # A serving batch, smaller blocks, gate and up pruned together.
        {"name": "gated_decode", "op": "gated", "tokens": 24, "cols": 4096, "rows": 12288, "block": 32, "keep": 0.25,
         "pattern": "shared", "act": "gelu_tanh", "dtype": "f16"},
        # Prompts packed into one batch at the linear-layer workload's widths.
        {"name": "gated_prompts", "op": "gated", "tokens": 8192, "cols": 8192, "rows": 32768, "block": 64, "keep": 0.2,
         "pattern": "shared", "act": "silu", "dtype": "bf16"},
        # A prompt of odd length through a half-dense layer pruned apart.
        {"name": "gated_prompt_odd", "op": "gated", "tokens": 1777, "cols": 4096, "rows": 11000, "block": 64,
         "keep": 0.5, "pattern": "own", "act": "gelu", "dtype": "f16"},
        # Training with an odd batch and widths that end inside a block.
        {"name": "gated_train_odd", "op": "gated_train", "tokens": 777, "cols": 1000, "rows": 520, "block": 64,
         "keep": 0.5, "pattern": "own", "act": "gelu", "dtype": "f16"},
        # Sparse training of a feed-forward block.
        {"name": "gated_train", "op": "gated_train", "tokens": 8192, "cols": 4096, "rows": 16384, "block": 64,
         "keep": 0.2, "pattern": "own", "act": "silu", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "loss_train", "loss_train", "gated", "gated", "gated_train"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    odd = rng.random() < 0.3
    if op in ("loss", "loss_train"):
        case = {"op": op, "vocab": _log(rng, 1000, 100000), "dim": _log(rng, 50, 3000) if odd else 64 * _log(rng, 1, 48),
                "tokens": _log(rng, 1, 6000), "dtype": dtype, "scale": rng.choice([1.0, 0.5]),
                "reduction": rng.choice(["mean", "sum", "none"])}
        return case
    case = {"op": op, "cols": _log(rng, 100, 6000) if odd else 64 * _log(rng, 4, 96),
            "rows": _log(rng, 100, 16000) if odd else 64 * _log(rng, 4, 256),
            "block": 64 if op == "gated_train" else rng.choice([32, 64, 64]), "keep": rng.choice([0.1, 0.2, 0.5, 0.9]),
            "pattern": rng.choice(["own", "shared"]), "act": rng.choice(["silu", "gelu", "gelu_tanh", "relu"]),
            "dtype": dtype}
    case["tokens"] = _log(rng, 1, 6000) if op == "gated" else _log(rng, 16, 6000)
    return case


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(std)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _mask(g, nbr, nbc, keep):
    """Positions of the kept blocks, ascending."""
    n = max(1, int(nbr * nbc * keep))
    return torch.sort(torch.randperm(nbr * nbc, generator=g, device="cuda")[:n]).values


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    s = {"case": case}
    t = case["tokens"]
    if case["op"] in ("loss", "loss_train"):
        v, d = case["vocab"], case["dim"]
        # Rows of norm 2 and hidden states of unit scale: logits of a spread of 2, and 4 to 8 more for the token that
        # follows, which a trained model knows about; some tokens are padding.
        s["weight"] = _randn(g, v, d, std=2.0 * d**-0.5, dtype=dt)
        ids = (v * _rand(g, t).double() ** _SKEW).long().clamp_(max=v - 1)
        known = (1.0 + _rand(g, t)[:, None]) / case["scale"]
        s["x"] = (_randn(g, t, d) + known * s["weight"][ids].float()).to(dt)
        s["targets"] = torch.where(_rand(g, t) < 0.05, -1, ids) if t > 8 else ids
        # the gradient by the loss: of one number, or of every token's
        s["grad"] = 0.5 + _rand(g, t) if case["reduction"] == "none" else 0.5 + _rand(g, 1)[0]
        return s
    bs, m, k = case["block"], case["rows"], case["cols"]
    nbr, nbc = -(-m // bs), -(-k // bs)
    s["x"] = _randn(g, t, k, dtype=dt)
    loud = _rand(g, k) < 0.002
    s["x"].mul_(torch.where(loud, 10.0, 1.0).to(dt))
    pos = _mask(g, nbr, nbc, case["keep"])
    for name in ("gate", "up"):
        if name == "up" and case["pattern"] == "own":
            pos = _mask(g, nbr, nbc, case["keep"])
        std = (case["keep"] * k) ** -0.5 * (2.0 if name == "gate" else 1.0)
        blocks = _randn(g, pos.numel(), bs, bs, std=std, dtype=dt)
        s[name] = {"blocks": blocks, "row": pos // nbc, "col": pos % nbc}
        # what a block has behind the matrix's last row or column is zero
        blocks.masked_fill_((s[name]["row"][:, None] * bs + torch.arange(bs, device="cuda") >= m)[:, :, None], 0.0)
        blocks.masked_fill_((s[name]["col"][:, None] * bs + torch.arange(bs, device="cuda") >= k)[:, None, :], 0.0)
    if case["op"] == "gated_train":
        s["dh"] = _randn(g, t, m, std=0.01, dtype=dt)
    if own:
        from kairo_b200.ops import bsr_from_tiles, gated_weights

        parts = [bsr_from_tiles(p["blocks"], p["row"].int(), p["col"].int(), (m, k)) for p in (s["gate"], s["up"])]
        s["weights"] = gated_weights(*parts)
    return s


# ---------------------------------------------------------------- plain forms


def _plain_loss(s):
    """Loss (reduced), lse, and the gradients by x and weight where the case trains."""
    case = s["case"]
    x, w, ids = s["x"].float(), s["weight"].float(), s["targets"]
    logits = (x @ w.t()).mul_(case["scale"])
    live = (ids >= 0) & (ids < case["vocab"])
    at = torch.where(live, ids, 0)[:, None]
    top = logits.amax(1, keepdim=True)
    target = logits.gather(1, at)
    logits.sub_(top).exp_()
    total = logits.sum(1, keepdim=True)
    lse = torch.log(total) + top
    each = torch.where(live, (lse - target)[:, 0], 0.0)
    count = live.sum().clamp(min=1)
    loss = {"none": each, "sum": each.sum(), "mean": each.sum() / count}[case["reduction"]]
    if case["op"] == "loss":
        return {"loss": loss, "lse": lse[:, 0]}
    factor = s["grad"] * live
    if case["reduction"] == "mean":
        factor = factor / count
    factor = factor[:, None] * case["scale"]
    logits.div_(total)  # the probabilities
    logits.scatter_add_(1, at, torch.full_like(target, -1.0))
    logits.mul_(factor)
    return {"loss": loss, "dx": (logits @ w).to(s["x"].dtype), "dw": (logits.t() @ x).to(s["x"].dtype)}


def _dense(p, m, k, bs):
    """A block-sparse matrix with zeros in its other blocks, in 32 bits, (m, k)."""
    nbr, nbc = -(-m // bs), -(-k // bs)
    out = torch.zeros(nbr, nbc, bs, bs, device="cuda")
    out[p["row"], p["col"]] = p["blocks"].float()
    return out.transpose(1, 2).reshape(nbr * bs, nbc * bs)[:m, :k]


def _blocks_of(dense, p, bs):
    """The blocks at p's places of a (m, k) matrix, zero behind its edges."""
    m, k = dense.shape
    full = torch.nn.functional.pad(dense, (0, -k % bs, 0, -m % bs))
    return full.view(full.shape[0] // bs, bs, full.shape[1] // bs, bs)[p["row"], :, p["col"], :]


def _plain_act(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-g))
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(g * -math.sqrt(0.5))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2.0 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        th = torch.tanh(c * (g + 0.044715 * g**3))
        return 0.5 * g * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * g * (1.0 - th * th) * c * (1.0 + 0.134145 * g * g)
    return g.clamp(min=0.0), (g > 0).float()


def _plain_gated(s):
    case = s["case"]
    m, k, bs, dt = case["rows"], case["cols"], case["block"], s["x"].dtype
    x = s["x"].float()
    wg, wu = (_dense(s[n], m, k, bs) for n in ("gate", "up"))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _plain_act(g, case["act"])
    h = (a * u).to(dt)
    if case["op"] == "gated":
        return h
    dh = s["dh"].float()
    dg, du = dh * u * da, dh * a
    return {"h": h, "dx": (dg @ wg + du @ wu).to(dt), "dgate": _blocks_of(dg.t() @ x, s["gate"], bs).to(dt),
            "dup": _blocks_of(du.t() @ x, s["up"], bs).to(dt)}


def _plain(s):
    return _plain_loss(s) if s["case"]["op"] in ("loss", "loss_train") else _plain_gated(s)


# ---------------------------------------------------------------- the framework's calls


def _own(s):
    from kairo_b200 import ops

    case = s["case"]
    if case["op"] in ("loss", "loss_train"):
        how = {"scale": case["scale"], "reduction": case["reduction"]}
        loss, lse = ops.linear_cross_entropy(s["x"], s["weight"], s["targets"], return_lse=True, **how)
        if case["op"] == "loss":
            return {"loss": loss, "lse": lse}
        dx, dw = ops.linear_cross_entropy_backward(s["grad"], s["x"], s["weight"], s["targets"], lse, **how)
        return {"loss": loss, "dx": dx, "dw": dw}
    h = ops.sparse_gated_linear(s["x"], s["weights"], activation=case["act"])
    if case["op"] == "gated":
        return h
    dx, dblocks = ops.sparse_gated_linear_backward(s["dh"], s["x"], s["weights"], activation=case["act"])
    dgate, dup = s["weights"].split(dblocks)
    return {"h": h, "dx": dx, "dgate": dgate, "dup": dup}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- the definition, in 64 bits


def _exact_loss(s):
    """One piece of the tokens after the other, by log_softmax."""
    case = s["case"]
    w, ids = s["weight"].double(), s["targets"]
    live = (ids >= 0) & (ids < case["vocab"])
    count = max(1, int(live.sum()))
    t = case["tokens"]
    each, lse = torch.zeros(2, t, dtype=torch.float64, device="cuda").unbind(0)
    dx = torch.zeros(t, case["dim"], dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(w)
    for at in torch.split(torch.arange(t, device="cuda"), 1024):
        x = s["x"][at].double()
        z = case["scale"] * (x @ w.t())
        lse[at] = torch.logsumexp(z, 1)
        rows = torch.nonzero(live[at])[:, 0]
        each[at[rows]] = lse[at[rows]] - z[rows, ids[at[rows]]]
        if case["op"] == "loss":
            continue
        p = torch.exp(z - lse[at][:, None])
        p[rows, ids[at[rows]]] -= 1.0
        weight = s["grad"][at].double() if case["reduction"] == "none" else s["grad"].double().expand(len(at))
        p *= (weight * live[at] * case["scale"] / (count if case["reduction"] == "mean" else 1))[:, None]
        dx[at] = p @ w
        dw += p.t() @ x
    loss = {"none": each, "sum": each.sum(), "mean": each.sum() / count}[case["reduction"]]
    return {"loss": loss, "lse": lse} if case["op"] == "loss" else {"loss": loss, "dx": dx, "dw": dw}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("loss", "loss_train"):
        return _exact_loss(s)
    m, k, bs = case["rows"], case["cols"], case["block"]
    x = torch.nn.functional.pad(s["x"].double(), (0, -k % bs))
    # block-row by block-row: the kept columns of x beside one another, times that row's blocks
    h = torch.zeros(case["tokens"], -(-m // bs) * bs, dtype=torch.float64, device="cuda")
    train = case["op"] == "gated_train"
    if train:
        dh = torch.nn.functional.pad(s["dh"].double(), (0, -m % bs))
        dx = torch.zeros_like(x)
        grads = {n: torch.zeros(s[n]["blocks"].shape, dtype=torch.float64, device="cuda") for n in ("gate", "up")}
    starts = {n: torch.searchsorted(s[n]["row"], torch.arange(-(-m // bs) + 1, device="cuda")).tolist()
              for n in ("gate", "up")}
    for i in range(-(-m // bs)):
        part = {}
        for n in ("gate", "up"):
            lo, hi = starts[n][i], starts[n][i + 1]
            cols = (s[n]["col"][lo:hi, None] * bs + torch.arange(bs, device="cuda")).flatten()
            w = s[n]["blocks"][lo:hi].double().transpose(0, 1).reshape(bs, -1)
            part[n] = (lo, hi, cols, w, x[:, cols] @ w.t())
        g = part["gate"][4].requires_grad_(train)
        a = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
             "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["act"]](g)
        at = slice(i * bs, (i + 1) * bs)
        h[:, at] = (a * part["up"][4]).detach()
        if train:
            d = {"gate": torch.autograd.grad(a, g, dh[:, at] * part["up"][4])[0], "up": dh[:, at] * a.detach()}
            for n in ("gate", "up"):
                lo, hi, cols, w, _ = part[n]
                dx[:, cols] += d[n] @ w
                grads[n][lo:hi] = (d[n].t() @ x[:, cols]).view(bs, hi - lo, bs).transpose(0, 1)
    if not train:
        return h[:, :m]
    return {"h": h[:, :m], "dx": dx[:, :k], "dgate": grads["gate"], "dup": grads["up"]}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    t = case["tokens"]
    if case["op"] in ("loss", "loss_train"):
        v, d = case["vocab"], case["dim"]
        both = 2 * (t + v) * d  # hidden states and table
        if case["op"] == "loss":
            return {"bytes": both + 16 * t, "flops": 2 * t * v * d}
        return {"bytes": 2 * both + 16 * t, "flops": 6 * t * v * d}
    bs, m, k = case["block"], case["rows"], case["cols"]
    blocks = 2 * max(1, int(-(-m // bs) * -(-k // bs) * case["keep"]))
    nbytes = 2 * (t * (m + k) + blocks * bs * bs)
    flops = 2 * t * blocks * bs * bs
    if case["op"] == "gated_train":
        return {"bytes": 2 * nbytes, "flops": 3 * flops}
    return {"bytes": nbytes, "flops": flops}
