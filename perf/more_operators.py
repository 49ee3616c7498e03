"""What stands between the aggregations of a deep graph network as measurable cases: the norm of its rows, dense layers with what follows them, and
8 bits a value for what either keeps for the backward pass.

``norm``: ``fastgl.layer_norm`` forward and backward, ``(x - mean) / sqrt(var + eps) * weight + bias`` over each row, negative values set to zero where
``relu``.  ``linear``: ``fastgl.linear`` forward and backward, ``activation(x W^T + b) + residual``.  ``keep8``: what the gradients of the weights (and
the norm's backward pass) take of the input is held in 8 bits: 32 neighbouring columns of a row share a step, the power of two ``2^(floor(log2(largest
magnitude)) - 6)``, and a value is the nearest of ``-127 .. 127`` steps; of the norm it is ``(x - mean) / sqrt(var + eps)`` that is held so.

Fields of a case: ``op``, ``dtype``, ``rows``, ``keep8``; norm: ``cols``, ``stride`` (of the rows), ``relu``; linear: ``dim``, ``out``, ``bias``,
``act``, ``residual``.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # -- the norm of the rows, forward and backward -------------------------------------------------------------
        # the smallest call: the hidden rows of an online batch
        dict(name="norm_small", op="norm", dtype="f32", rows=1024, cols=47, stride=47, relu=False, keep8=False),
        # hidden rows of a batch of 8192, the activation with it
        dict(name="norm_hidden", op="norm", dtype="f32", rows=60_000, cols=256, stride=256, relu=True, keep8=False),
        # the same in bf16, kept in 8 bits
        dict(name="norm_hidden_bf16_keep8", op="norm", dtype="bf16", rows=87_000, cols=256, stride=256, relu=True, keep8=True),
        # a whole graph's rows, columns of a wider table, kept in 8 bits
        dict(name="norm_graph_keep8", op="norm", dtype="f32", rows=2_400_000, cols=64, stride=100, relu=False, keep8=True),
        # features as they come, an odd number of rows
        dict(name="norm_features_bf16", op="norm", dtype="bf16", rows=200_003, cols=602, stride=602, relu=False, keep8=False),
        # -- dense layers, forward and backward -----------------------------------------------------------------------
        # a handful of seeds
        dict(name="linear_small", op="linear", dtype="f32", rows=100, dim=64, out=47, bias=True, act=None, residual=False, keep8=False),
        # a layer with a residual over a batch's hidden rows
        dict(name="linear_residual", op="linear", dtype="f32", rows=60_000, dim=256, out=256, bias=True, act="gelu", residual=True, keep8=False),
        # features to hidden rows, the features kept in 8 bits
        dict(name="linear_features_keep8", op="linear", dtype="f32", rows=107_000, dim=100, out=256, bias=True, act="silu", residual=False, keep8=True),
        dict(name="linear_wide_keep8", op="linear", dtype="f32", rows=8192, dim=602, out=256, bias=True, act=None, residual=False, keep8=True),
        # a feed-forward block's two layers in bf16: up with an activation, down with the residual
        dict(name="linear_up_bf16", op="linear", dtype="bf16", rows=87_000, dim=256, out=512, bias=True, act="relu", residual=False, keep8=False),
        dict(name="linear_down_bf16_keep8", op="linear", dtype="bf16", rows=87_000, dim=512, out=256, bias=True, act=None, residual=True, keep8=True),
        # a whole graph's rows through a narrow layer
        dict(name="linear_graph_bf16", op="linear", dtype="bf16", rows=2_400_000, dim=100, out=64, bias=False, act="silu", residual=False, keep8=False),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    dtype = rng.choice(["f32", "bf16"])
    if rng.random() < 0.45:
        cols = rng.choice([_log_uniform(rng, 8, 1024), rng.randint(16, 602), 64, 128, 256])
        rows = _log_uniform(rng, 1, 120_000_000 // max(cols, 64))
        return dict(op="norm", dtype=dtype, rows=rows, cols=cols, stride=cols + rng.choice([0, 0, rng.randint(1, 64)]), relu=rng.random() < 0.5,
                    keep8=rng.random() < 0.5)
    dim = rng.choice([_log_uniform(rng, 8, 1024), rng.randint(16, 602), 64, 128, 256])
    out = rng.choice([_log_uniform(rng, 8, 1024), rng.randint(16, 512), 64, 128, 256, 512])
    rows = _log_uniform(rng, 1, min(2_400_000, 11_000_000_000 // (dim * out), 150_000_000 // max(dim, out, 64)))
    # (in fp32 no step in a derivative: a sum that rounds to the other side of it is another gradient, whoever formed it)
    return dict(op="linear", dtype=dtype, rows=rows, dim=dim, out=out, bias=rng.random() < 0.7, act=rng.choice([None, "gelu", "silu", "silu" if dtype == "f32" else "relu"]),
                residual=rng.random() < 0.4, keep8=rng.random() < 0.5)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    normal = lambda *size: torch.randn(size, generator=gen, device=DEV)  # noqa: E731
    s = dict(case)
    n = case["rows"]
    if case["op"] == "norm":
        d = case["cols"]
        # rows of different means and sizes, as sums over neighbours are
        x = normal(n, case["stride"]) * (0.25 + 2 * torch.rand((n, 1), generator=gen, device=DEV)) + normal(n, 1)
        s["x"] = x.to(dtype)[:, :d].requires_grad_()
        s["weight"] = (1 + 0.2 * normal(d)).to(dtype).requires_grad_()
        s["bias"] = (0.2 * normal(d)).to(dtype).requires_grad_()
        s["d_out"] = normal(n, d).to(dtype)
        return s
    k, m = case["dim"], case["out"]
    s["x"] = normal(n, k).to(dtype).requires_grad_()
    s["weight"] = (normal(m, k) / k ** 0.5).to(dtype).requires_grad_()
    s["bias"] = (0.2 * normal(m)).to(dtype).requires_grad_() if case["bias"] else None
    s["residual"] = normal(n, m).to(dtype).requires_grad_() if case["residual"] else None
    s["d_out"] = normal(n, m).to(dtype)
    return s


# -- in plain operations ------------------------------------------------------------------------------------------------
def _in_8_bits(v):
    """What 8 bits a value hold of the rows ``v``."""
    n, d = v.shape
    wide = -(-d // 32) * 32
    g = v.new_zeros((n, wide))
    g[:, :d] = v
    g = g.view(n, wide // 32, 32)
    exponent = torch.frexp(g.abs().amax(2, keepdim=True))[1].clamp(min=-119) - 7
    g = torch.ldexp(torch.ldexp(g, -exponent).round().clamp(-127, 127), exponent)
    return g.view(n, wide)[:, :d]


def _norm(s):
    # (64 bits for what says which values are cut to zero and which step one is nearest to)
    x, w, b, dy = s["x"].detach(), s["weight"].detach().float(), s["bias"].detach().float(), s["d_out"].float()
    wide = x.double()
    wide = wide - wide.mean(1, keepdim=True)
    scale = (wide.square().mean(1, keepdim=True) + EPS).rsqrt()
    wide = wide * scale
    h, scale = wide.float(), scale.float()
    y = h * w + b
    if s["relu"]:
        positive = wide * w.double() + b.double() > 0
        zero = torch.zeros((), device=DEV)
        y, dy = torch.where(positive, y, zero), torch.where(positive, dy, zero)
    if s["keep8"]:
        h = _in_8_bits(wide).float()
    del wide
    d_w, d_b = (dy * h).sum(0), dy.sum(0)
    g = dy * w
    d_x = (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) * scale
    return [t.to(x.dtype) for t in (y, d_x, d_w, d_b)]


def _activation(z, act):
    """The activation of ``z`` and its derivative (None: one)."""
    if act == "relu":
        return z.clamp(min=0), (z > 0).float()
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    return z, None


def _linear(s):
    dtype = s["x"].dtype
    x, w, dy = s["x"].detach().float(), s["weight"].detach().float(), s["d_out"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    y, slope = _activation(z, s["act"])
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    dz = dy if slope is None else dy * slope
    if s["keep8"]:
        x = _in_8_bits(x)
    out = [y, dz @ w, dz.t() @ x]
    if s["bias"] is not None:
        out.append(dz.sum(0))
    if s["residual"] is not None:
        out.append(dy)
    return [t.to(dtype) for t in out]


def run(state):
    s = state
    if own:
        at = os.path.join(os.getcwd(), "fastgl-ae_amd")  # the repository's root is the working folder
        if at not in sys.path:
            sys.path.insert(0, at)
        import fastgl

        if s["op"] == "norm":
            y = fastgl.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, relu=s["relu"], keep8=s["keep8"])
            of = [s[k] for k in ("x", "weight", "bias")]
        else:
            y = fastgl.linear(s["x"], s["weight"], s["bias"], activation=s["act"], residual=s["residual"], keep8=s["keep8"])
            of = [s[k] for k in ("x", "weight", "bias", "residual") if s[k] is not None]
        return [y.detach(), *torch.autograd.grad(y, of, s["d_out"])]
    return _norm(s) if s["op"] == "norm" else _linear(s)


def work(case):
    size, n = 4 if case["dtype"] == "f32" else 2, case["rows"]
    if case["op"] == "norm":
        # x, the output's gradient and the parameters in, the output and three gradients out; about twenty operations a value
        return dict(bytes=size * (4 * n * case["cols"] + 4 * case["cols"]), flops=20 * n * case["cols"])
    k, m = case["dim"], case["out"]
    return dict(bytes=size * (2 * n * k + 2 * n * m + 2 * m * k + (2 * m if case["bias"] else 0) + (2 * n * m if case["residual"] else 0)), flops=6 * n * k * m)


# -- 64 bits ------------------------------------------------------------------------------------------------------------
def _held(v):
    """The nearest multiples of each 32 columns' step, in 64 bits."""
    out = torch.empty_like(v)
    for c in range(0, v.size(1), 32):
        part = v[:, c:c + 32]
        top = part.abs().max(1, keepdim=True).values
        power = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
        power = torch.where(torch.exp2(power) > top, power - 1, torch.where(torch.exp2(power + 1) <= top, power + 1, power))
        step = torch.exp2(torch.where(top > 0, power, torch.full_like(top, -120.0)).clamp(min=-120) - 6)
        out[:, c:c + 32] = torch.minimum(torch.maximum(torch.round(part / step), torch.full_like(part, -127.0)), torch.full_like(part, 127.0)) * step
    return out


def _exact_norm(case, s):
    x, w, b = s["x"].detach(), s["weight"].detach().double(), s["bias"].detach().double()
    n, d = x.shape
    y, d_x = torch.empty((n, d), dtype=torch.float64, device=DEV), torch.empty((n, d), dtype=torch.float64, device=DEV)
    d_w, d_b = torch.zeros_like(w), torch.zeros_like(b)
    step = max(1, 40_000_000 // d)
    for first in range(0, n, step):
        rows = slice(first, min(n, first + step))
        r, g = x[rows].double(), s["d_out"][rows].double()
        var, mean = torch.var_mean(r, 1, unbiased=False, keepdim=True)
        sigma = torch.sqrt(var + EPS)
        h = (r - mean) / sigma
        out = torch.addcmul(b, h, w)
        if case["relu"]:
            g = g * (out > 0)
            out = out.relu()
        y[rows] = out
        if case["keep8"]:
            h = _held(h)
        d_w += torch.einsum("rc,rc->c", g, h)
        d_b += g.sum(0)
        g = g * w
        d_x[rows] = (g - (g.sum(1, keepdim=True) + h * (g * h).sum(1, keepdim=True)) / d) / sigma
    return [y, d_x, d_w, d_b]


def _exact_linear(case, s):
    x, w = s["x"].detach(), s["weight"].detach().double()
    n, m = x.size(0), w.size(0)
    y, d_x = torch.empty((n, m), dtype=torch.float64, device=DEV), torch.empty(x.shape, dtype=torch.float64, device=DEV)
    d_w, d_b = torch.zeros_like(w), torch.zeros(m, dtype=torch.float64, device=DEV)
    step = max(1, 40_000_000 // max(m, x.size(1)))
    for first in range(0, n, step):
        rows = slice(first, min(n, first + step))
        r, g = x[rows].double(), s["d_out"][rows].double()
        z = r @ w.t() if s["bias"] is None else torch.addmm(s["bias"].detach().double(), r, w.t())
        if case["act"] == "relu":
            out, g = z.relu(), g * (z > 0)
        elif case["act"] == "silu":
            p = torch.sigmoid(z)
            out, g = z * p, g * (p + z * p * torch.sigmoid(-z))
        elif case["act"] == "gelu":
            p = 0.5 * torch.erfc(-z / math.sqrt(2))
            out, g = z * p, g * (p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
        else:
            out = z
        y[rows] = out if s["residual"] is None else out + s["residual"].detach()[rows].double()
        d_x[rows] = g @ w
        d_w += g.t() @ (_held(r) if case["keep8"] else r)
        d_b += g.sum(0)
    return [y, d_x, d_w] + ([] if s["bias"] is None else [d_b]) + ([] if s["residual"] is None else [s["d_out"].double()])


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(case, s) if case["op"] == "norm" else _exact_linear(case, s)
