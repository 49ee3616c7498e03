"""The two ends of a training step as measurable cases: the dropout between layers and the loss over the classes.

``dropout``: ``fastgl.dropout`` forward and backward, element ``i`` (row-major) kept where word ``i % 4`` of Philox4x32-10 with
counter ``(i // 4 low, i // 4 high, stream, 0x44524F50)`` and key ``seed`` is at least ``round(p * 2**32)``.
``xent``: ``fastgl.linear_cross_entropy``, softmax cross entropy of ``x W^T + b`` with the gradients of all three, or the losses alone.

Fields of a case: ``op``, ``dtype``; dropout: ``rows``, ``cols``, ``stride`` (of the rows), ``p``, ``relu``; xent: ``rows``, ``dim``,
``classes``, ``bias``, ``ignored`` (the share of rows without a label), ``reduction``, ``grad``.
"""
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
IGNORE = -100
TAG = 0x44524F50


def listed():
    return [
        # -- dropout between layers, forward and backward ---------------------------------------------------------
        # the smallest call: the hidden rows of an online batch
        dict(name="dropout_small", op="dropout", dtype="f32", rows=1024, cols=47, stride=47, p=0.5, relu=False),
        # GCN's hidden rows of a batch of 8192
        dict(name="dropout_gcn", op="dropout", dtype="f32", rows=60_000, cols=256, stride=256, p=0.5, relu=False),
        # GraphSAGE in bf16: activation and dropout of the first layer's rows
        dict(name="dropout_sage_bf16", op="dropout", dtype="bf16", rows=87_000, cols=256, stride=256, p=0.5, relu=True),
        # a whole graph's rows, columns of a wider table
        dict(name="dropout_graph", op="dropout", dtype="f32", rows=2_400_000, cols=64, stride=100, p=0.1, relu=False),
        # -- the loss and its gradients ---------------------------------------------------------------------------
        # a handful of seeds
        dict(name="xent_small", op="xent", dtype="f32", rows=100, dim=64, classes=47, bias=True, ignored=0.0, reduction="mean", grad=True),
        # node classification, a full batch, seeds without a label among it
        dict(name="xent_classes_bf16", op="xent", dtype="bf16", rows=8192, dim=256, classes=47, bias=True, ignored=0.3, reduction="mean", grad=True),
        dict(name="xent_classes", op="xent", dtype="f32", rows=8192, dim=256, classes=172, bias=True, ignored=0.0, reduction="mean", grad=True),
        # one entity out of all: link prediction against every node of a small graph
        dict(name="xent_entities_bf16", op="xent", dtype="bf16", rows=8192, dim=256, classes=100_000, bias=False, ignored=0.0, reduction="mean", grad=True),
        dict(name="xent_entities", op="xent", dtype="f32", rows=8192, dim=128, classes=20_011, bias=True, ignored=0.1, reduction="mean", grad=True),
        # the same for evaluation: each row's loss, no gradients
        dict(name="xent_rank_bf16", op="xent", dtype="bf16", rows=2000, dim=100, classes=100_003, bias=True, ignored=0.0, reduction="none", grad=False),
        # rows of eight attention heads of 64 columns, weighted one by one
        dict(name="xent_wide_bf16", op="xent", dtype="bf16", rows=1000, dim=512, classes=10_007, bias=False, ignored=0.0, reduction="none", grad=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    dtype = rng.choice(["f32", "bf16"])
    if rng.random() < 0.35:
        cols = rng.choice([rng.randint(1, 602), 64, 128, 256])
        rows = _log_uniform(rng, 1, 150_000_000 // max(cols, 64))
        return dict(op="dropout", dtype=dtype, rows=rows, cols=cols, stride=cols + rng.choice([0, 0, rng.randint(1, 64)]), p=round(rng.uniform(0.05, 0.9), 3),
                    relu=rng.random() < 0.5)
    rows = rng.choice([_log_uniform(rng, 1, 8192), 1000, 2000, 8192])
    dim = rng.choice([_log_uniform(rng, 8, 512), rng.randint(16, 256), 64, 128, 256])
    most = min(100_000, (200_000_000_000 if dtype == "bf16" else 20_000_000_000) // (rows * dim))
    grad = rng.random() < 0.8
    return dict(op="xent", dtype=dtype, rows=rows, dim=dim, classes=_log_uniform(rng, 2, max(most, 4)), bias=rng.random() < 0.6,
                ignored=rng.choice([0.0, 0.0, 0.1, 0.5]), reduction=rng.choice(["mean", "mean", "sum", "none"]), grad=grad)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    normal = lambda *size: torch.randn(size, generator=gen, device=DEV)  # noqa: E731
    s = dict(case)
    if case["op"] == "dropout":
        rows, cols = case["rows"], case["cols"]
        s["x"] = normal(rows, case["stride"]).to(dtype)[:, :cols].requires_grad_()
        s["d_out"] = normal(rows, cols).to(dtype)
        s["seed"], s["stream"] = seed * 0x9E3779B97F4A7C15 % 2 ** 64, seed % 1000
        return s
    n, d, v = case["rows"], case["dim"], case["classes"]
    # a model on its way: rows that are certain of their class and rows that are not
    w = normal(v, d) / d ** 0.5
    y = torch.randint(0, v, (n,), generator=gen, device=DEV)
    x = normal(n, d) + w.index_select(0, y) * (8 * torch.rand((n, 1), generator=gen, device=DEV))
    if case["ignored"]:
        y = torch.where(torch.rand(n, generator=gen, device=DEV) < case["ignored"], torch.full_like(y, IGNORE), y)
        y[0] = 0
    s["x"], s["weight"], s["labels"] = x.to(dtype), w.to(dtype), y
    s["bias"] = normal(v).to(dtype) if case["bias"] else None
    if case["grad"]:
        for k in ("x", "weight", "bias"):
            if s[k] is not None:
                s[k].requires_grad_()
    s["d_loss"] = torch.rand(n if case["reduction"] == "none" else (), generator=gen, device=DEV) + 0.5
    return s


# -- dropout ----------------------------------------------------------------------------------------------------------
def _kept(n, p, seed, stream):
    """Which of the elements 0 .. n - 1 are kept, by the generator's rounds on whole numbers."""
    low = 0xFFFFFFFF
    quad = torch.arange((n + 3) // 4, device=DEV)
    c0, c1, c2, c3 = quad & low, quad >> 32, torch.full_like(quad, stream & low), torch.full_like(quad, TAG)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (modulo 2^64: the two halves are the product's)
        c0, c1, c2, c3 = (b >> 32) & low ^ c1 ^ k0, b & low, (a >> 32) & low ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:n]
    return words >= round(p * 2.0 ** 32)


def _dropout(s):
    x, d_out = s["x"].detach(), s["d_out"]
    kept = _kept(x.numel(), s["p"], s["seed"], s["stream"]).view(x.shape)
    scale = 1.0 / (1.0 - s["p"])
    value = x.float()
    if s["relu"]:
        kept = kept & (value > 0)
    zero = torch.zeros((), device=DEV)
    return torch.where(kept, value * scale, zero).to(x.dtype), torch.where(kept, d_out.float() * scale, zero).to(x.dtype)


# -- the loss ---------------------------------------------------------------------------------------------------------
def _xent(s):
    x, w, y = s["x"].detach().float(), s["weight"].detach().float(), s["labels"]
    valid = y != IGNORE
    label = torch.where(valid, y, torch.zeros_like(y))[:, None]
    logits = x @ w.t()
    if s["bias"] is not None:
        logits = logits + s["bias"].detach().float()
    top = logits.amax(1, keepdim=True)
    below = (top - logits.gather(1, label))[:, 0]
    p = torch.exp(logits - top)
    del logits
    of_label = p.gather(1, label)[:, 0]
    others = p.scatter_(1, label, 0.0).sum(1)  # (without the label's: one minus its probability loses no bits)
    total = others + of_label
    zero = torch.zeros((), device=DEV)
    losses = torch.where(below < 64, torch.log1p(others / of_label), torch.log(total) + below)
    losses = torch.where(valid, losses, zero)
    count = valid.sum()
    loss = losses if s["reduction"] == "none" else losses.sum() if s["reduction"] == "sum" else losses.sum() / count
    if not s["grad"]:
        return [loss]
    g = torch.where(valid, s["d_loss"] if s["reduction"] != "mean" else s["d_loss"] / count, zero)
    p = p.scatter_(1, label, -others[:, None]) * (g / total)[:, None]
    out = [loss, (p @ w).to(s["x"].dtype), (p.t() @ x).to(s["x"].dtype)]
    if s["bias"] is not None:
        out.append(p.sum(0).to(s["x"].dtype))
    return out


def run(state):
    s = state
    if own:
        at = os.path.join(os.getcwd(), "fastgl-ae_amd")  # the repository's root is the working folder
        if at not in sys.path:
            sys.path.insert(0, at)
        import fastgl

        if s["op"] == "dropout":
            y = fastgl.dropout(s["x"], s["p"], seed=s["seed"], stream=s["stream"], relu=s["relu"])
            return [y.detach(), torch.autograd.grad(y, s["x"], s["d_out"])[0]]
        loss = fastgl.linear_cross_entropy(s["x"], s["weight"], s["labels"], s["bias"], ignore_index=IGNORE, reduction=s["reduction"])
        if not s["grad"]:
            return [loss]
        of = [s[k] for k in ("x", "weight", "bias") if s[k] is not None]
        return [loss.detach(), *torch.autograd.grad(loss, of, s["d_loss"])]
    return list(_dropout(s)) if s["op"] == "dropout" else _xent(s)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        # x and the output's gradient in, the output and x's gradient out; ten rounds of two products and six other operations for four elements
        return dict(bytes=4 * n * size, flops=2 * n)
    n, d, v = case["rows"], case["dim"], case["classes"]
    inputs = size * (n * d + v * d + (v if case["bias"] else 0)) + 8 * n
    losses = 4 * (n if case["reduction"] == "none" else 1)
    if not case["grad"]:
        return dict(bytes=inputs + losses, flops=2 * n * v * d)
    return dict(bytes=inputs + 2 * losses + size * (n * d + v * d + (v if case["bias"] else 0)), flops=6 * n * v * d)


# -- 64 bits ----------------------------------------------------------------------------------------------------------
def _product32(a, m):
    """The low and the high 32 bits of a * m, by halves of 16 bits."""
    a0, a1, m0, m1 = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
    low = a0 * m0
    mid = a1 * m0 + (low >> 16)
    more = a0 * m1 + (mid & 0xFFFF)
    return ((more & 0xFFFF) << 16) | (low & 0xFFFF), a1 * m1 + (mid >> 16) + (more >> 16)


def _exact_dropout(case, s):
    x = s["x"].detach()
    n = x.numel()
    keep = torch.empty(n, dtype=torch.bool, device=DEV)
    step = 1 << 24
    for first in range(0, n, step):
        i = torch.arange(first, min(n, first + step), device=DEV)
        word = i % 4
        c = [i // 4 % 2 ** 32, i // 4 // 2 ** 32, torch.full_like(i, s["stream"]), torch.full_like(i, TAG)]
        key = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32]
        for _ in range(10):
            lo0, hi0 = _product32(c[0], 0xD2511F53)
            lo1, hi1 = _product32(c[2], 0xCD9E8D57)
            c = [hi1 ^ c[1] ^ key[0], lo1, hi0 ^ c[3] ^ key[1], lo0]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        r = c[3]
        for k in range(3):
            r = torch.where(word == k, c[k], r)
        keep[first:first + i.numel()] = r.double() / 2.0 ** 32 >= round(case["p"] * 2.0 ** 32) / 2.0 ** 32
    keep = keep.view(x.shape)
    if case["relu"]:
        keep = keep & (x > 0)
    share = keep.double() / (1.0 - case["p"])
    return [x.double() * share, s["d_out"].double() * share]


def _exact_xent(case, s):
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    b = torch.zeros(case["classes"], dtype=torch.float64, device=DEV) if s["bias"] is None else s["bias"].detach().double()
    y = s["labels"]
    count = int((y != IGNORE).sum())
    losses = torch.zeros(case["rows"], dtype=torch.float64, device=DEV)
    d_x, d_w, d_b = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    step = max(1, 200_000_000 // case["classes"])
    for first in range(0, case["rows"], step):
        rows = torch.arange(first, min(case["rows"], first + step), device=DEV)
        rows = rows[y[rows] != IGNORE]
        if rows.numel() == 0:
            continue
        log_p = torch.addmm(b, x[rows], w.t())
        log_p -= torch.logsumexp(log_p, 1, keepdim=True)
        at = torch.arange(rows.numel(), device=DEV)
        losses[rows] = -log_p[at, y[rows]]
        if not case["grad"]:
            continue
        d = log_p.exp_()
        d[at, y[rows]] = torch.expm1(-losses[rows])
        d *= s["d_loss"].double()[rows, None] if case["reduction"] == "none" else s["d_loss"].double() / (count if case["reduction"] == "mean" else 1)
        d_x[rows] = d @ w
        d_w += d.t() @ x[rows]
        d_b += d.sum(0)
    loss = losses if case["reduction"] == "none" else losses.sum() / (count if case["reduction"] == "mean" else 1)
    return [loss] if not case["grad"] else [loss, d_x, d_w] + ([] if s["bias"] is None else [d_b])


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_dropout(case, s) if case["op"] == "dropout" else _exact_xent(case, s)
