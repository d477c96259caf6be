"""Workloads of the operators of a window transformer block in its plain form, next to this framework's modulated one: layer
norm, a linear layer with bias, activation and residual, and attention in windows with a learned bias by relative position
(buckets), each forward and backward.

    listed()            the fixed cases
    draw(rng)           one more case from the ranges the fixed ones stand for
    prepare(case, seed) inputs on the GPU
    run(state)          one pass, in the operators' plain form or, where ``own`` is set, through the framework's entry points
    work(case)          bytes and floating-point operations that one pass cannot do without
    exact(case, seed)   what ``run`` returns, computed in 64 bits

Kinds of case: ``ln`` (layer norm), ``ln-grad`` (its gradients), ``lin`` (linear layer), ``lin-grad`` (its gradients), ``attn``
(attention with a position bias) and ``attn-grad`` (its gradients, those of the bias table among them).
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
LOG2E = 1.4426950408889634
HIDDEN = -1e30         # an entry of the bias table that is no larger hides the pairs of its bucket


# ------------------------------------------------------------------------------------------------------------ cases
def _ln(kind: str, rows: int, cols: int, dtype: str = "bfloat16", affine: bool = True, pitch: int = 0) -> dict:
    """``pitch``: elements that rows of x lie further apart than ``cols`` (x is a section of a wider matrix)."""
    return dict(kind=kind, rows=rows, cols=cols, dtype=dtype, affine=affine, pitch=pitch)


def _lin(kind: str, rows: int, inner: int, cols: int, act: str, bias: bool = True, resid: bool = False, keep: bool = False) -> dict:
    """x [rows, inner] -> [rows, cols]; ``keep``: the values before the activation are an output too (a training step)."""
    return dict(kind=kind, rows=rows, inner=inner, cols=cols, act=act, bias=bias, resid=resid, keep=keep)


def _attn(kind: str, windows: int, high: int, wide: int, heads: int, head_dim: int, coarse: bool = False, reach: int = 0) -> dict:
    """Windows of ``high`` x ``wide`` tokens. ``coarse``: distances share buckets whose width grows with the distance, else
    every relative position is a bucket of its own; ``reach``: positions further apart than this along an axis do not see each
    other (0: all do)."""
    return dict(kind=kind, windows=windows, high=high, wide=wide, heads=heads, head_dim=head_dim, coarse=coarse, reach=reach)


def listed() -> list[dict]:
    cases = {
        # one token of the flagship's 1536 channels: nothing but latency
        "ln-one-token": _ln("ln", 1, 1536),
        # a chunk of 72 windows of 900 tokens of the flagship
        "ln-chunk": _ln("ln", 64800, 1536),
        # odd sizes in fp32, out of a wider matrix
        "ln-grad-odd": _ln("ln-grad", 12345, 1001, "float32", pitch=3),
        # the gradients of the flagship's chunk, sums over 64,800 rows among them
        "ln-grad-chunk": _ln("ln-grad", 64800, 1536),
        # one token through the flagship's first MLP matrix
        "lin-one-token": _lin("lin", 1, 1536, 4096, "gelu"),
        # the flagship's chunk through it in training: the values before the activation are kept
        "lin-chunk": _lin("lin", 64800, 1536, 4096, "gelu", keep=True),
        # odd sizes: nothing is a multiple of anything
        "lin-grad-odd": _lin("lin-grad", 1111, 333, 777, "silu"),
        # gradients of a medium model's MLP matrix
        "lin-grad-medium": _lin("lin-grad", 28800, 768, 2048, "gelu_tanh"),
        # a toy model's windows: 16 of 8 x 8 tokens, two heads of 32
        "attn-toy": _attn("attn", 16, 8, 8, 2, 32),
        # a chunk of the flagship's windows of 30 x 30 tokens, 24 heads of 64
        "attn-chunk": _attn("attn", 72, 30, 30, 24, 64),
        # gradients in odd windows, shared buckets and positions that do not see each other, narrow heads
        "attn-grad-odd": _attn("attn-grad", 50, 9, 13, 5, 40, coarse=True, reach=7),
        # and of the flagship's chunk
        "attn-grad-chunk": _attn("attn-grad", 72, 30, 30, 24, 64),
    }
    return [{"name": name, **c} for name, c in cases.items()]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["ln", "ln-grad", "lin", "lin-grad", "attn", "attn-grad"])
    if kind.startswith("ln"):
        cols = _log_int(rng, 16, 16384)
        rows = _log_int(rng, 1, min(100000, 64800 * 1536 // cols))
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        if dtype == "float32":
            rows = max(1, rows // 2)
        return _ln(kind, rows, cols, dtype, rng.random() < 0.8, rng.choice([0, 0, 1, 8, 24]))
    if kind.startswith("lin"):
        inner, cols = _log_int(rng, 1, 5120), _log_int(rng, 1, 5120)
        if rng.random() < 0.6:
            inner, cols = (max(64, n // 64 * 64) for n in (inner, cols))
        most = 64800 * 1536 * 4096 // (inner * cols * (2 if kind == "lin-grad" else 1))
        rows = _log_int(rng, 1, max(1, min(64800, most)))
        act = rng.choice(["none", "gelu", "gelu_tanh", "relu", "silu"])
        bias, resid, keep = rng.random() < 0.8, rng.random() < 0.4, rng.random() < 0.4
        return _lin(kind, rows, inner, cols, act, bias, resid and kind == "lin", keep and kind == "lin" and act != "none")
    high, wide = _log_int(rng, 1, 40), _log_int(rng, 1, 40)
    d = rng.choice([16, 24, 32, 40, 64, 64, 64, 72, 96, 128, 128])
    heads = rng.choice([1, 2, 3, 4, 5, 6, 8, 12, 16, 24])
    if high * wide == 1:
        wide = 2
    n = high * wide
    most = min(72 * 24 * 900 ** 2 // (heads * n * n), 64800 * 24 * 64 // (heads * n * d))
    windows = _log_int(rng, 1, max(1, min(2000, most)))
    coarse = rng.random() < 0.4
    return _attn(kind, windows, high, wide, heads, d, coarse, rng.choice([0, 0, 0, _log_int(rng, 1, 40)]))


# ------------------------------------------------------------------------------------------------------------ inputs
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(1000003 * seed + 29)


def _steps(n: int, coarse: bool, reach: int) -> tuple[list[int], int]:
    """Bucket of every distance -(n - 1) .. n - 1 along one axis, and how many there are; ``reach``: those further are bucket 0."""
    def bucket(x: int) -> int:
        a = abs(x)
        if reach and a > reach:
            return 0
        if coarse and a > 4:
            a = 4 + int(2 * math.log2(a / 4))
        return 1 + 2 * a - (x > 0)
    got = [bucket(x) for x in range(1 - n, n)]
    return got, max(got) + 1


def prepare(case: dict, seed: int) -> dict:
    c, g = case, _generator(seed)
    s = {"case": c}
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)  # noqa: E731
    if c["kind"].startswith("ln"):
        dt, rows, cols = getattr(torch, c["dtype"]), c["rows"], c["cols"]
        wide = torch.empty((rows, cols + c["pitch"]), dtype=dt, device=DEVICE)
        s["x"] = wide[:, :cols]
        # a stream whose rows differ in strength and mean
        s["x"].copy_(normal(rows, cols) * (0.5 + normal(rows, 1).abs()) + 0.3 * normal(rows, 1))
        s["w"] = (1 + 0.2 * normal(cols)).to(dt) if c["affine"] else None
        s["b"] = (0.1 * normal(cols)).to(dt) if c["affine"] else None
        if c["kind"] == "ln-grad":
            s["dy"] = (0.01 * normal(rows, cols)).to(dt)
            x = s["x"].double()
            mean = x.mean(1)
            s["stats"] = torch.stack([mean, ((x - mean[:, None]).square().mean(1) + EPS).rsqrt()], 1).float()
        return s
    if c["kind"].startswith("lin"):
        rows, inner, cols = c["rows"], c["inner"], c["cols"]
        s["x"] = normal(rows, inner).bfloat16()
        s["w"] = (normal(cols, inner) / math.sqrt(inner)).bfloat16()
        s["b"] = 0.2 * normal(cols) if c["bias"] else None
        s["resid"] = normal(rows, cols).bfloat16() if c["resid"] else None
        if c["kind"] == "lin-grad":
            s["dy"] = (0.01 * normal(rows, cols)).bfloat16()
            s["z"] = None
            if c["act"] != "none":
                z = s["x"].float() @ s["w"].float().T
                s["z"] = (z if s["b"] is None else z + s["b"]).bfloat16()
        return s
    n, heads, d, h, w = c["high"] * c["wide"], c["heads"], c["head_dim"], c["high"], c["wide"]
    s["qkv"] = normal(c["windows"] * n, 3 * heads * d).bfloat16()
    if c["coarse"] or c["reach"]:
        (by, ny), (bx, nx) = _steps(h, c["coarse"], c["reach"]), _steps(w, c["coarse"], c["reach"])
        # bucket 0: not seen along one axis or the other
        b = [[1 + (y - 1) * nx + (x - 1) if x and y else 0 for x in bx] for y in by]
        s["buckets"] = torch.tensor(b, dtype=torch.int32, device=DEVICE).reshape(-1)
        s["table"] = 0.8 * normal(1 + ny * nx, heads)
        s["table"][0] = -math.inf
    else:
        s["buckets"] = None
        s["table"] = 0.8 * normal((2 * h - 1) * (2 * w - 1), heads)
    if c["kind"] == "attn-grad":
        s["d_o"] = (0.1 * normal(c["windows"] * n, heads * d)).bfloat16()
        o, s["lse"] = _plain_attn(s)
        s["o"] = o.bfloat16()
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _plain_ln(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    y = x - mean
    rstd = torch.rsqrt(y.square().mean(1, keepdim=True) + EPS)
    y = y * rstd
    if s["w"] is not None:
        y = y * s["w"].float() + s["b"].float()
    return y.to(s["x"].dtype), torch.cat([mean, rstd], 1)


def _plain_ln_grad(s):
    mean, rstd = s["stats"][:, :1], s["stats"][:, 1:]
    dy, xhat = s["dy"].float(), (s["x"].float() - mean) * rstd
    g = dy if s["w"] is None else dy * s["w"].float()
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    dx = dx.to(s["x"].dtype)
    return dx if s["w"] is None else (dx, (dy * xhat).sum(0), dy.sum(0))


def _cdf(z):
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))


def _plain_act(z, act: str):
    if act == "gelu":
        return z * _cdf(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z.clamp_min(0) if act == "relu" else z


def _plain_act_grad(z, act: str):
    if act == "gelu":
        return _cdf(z) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * (math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z))
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return (z > 0).float()


def _plain_lin(s):
    z = s["x"].float() @ s["w"].float().T
    if s["b"] is not None:
        z = z + s["b"]
    y = _plain_act(z, s["case"]["act"])
    if s["resid"] is not None:
        y = s["resid"].float() + y
    return (y.bfloat16(), z.bfloat16()) if s["case"]["keep"] else y.bfloat16()


def _plain_lin_grad(s):
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = dz * _plain_act_grad(s["z"].float(), s["case"]["act"])
    dx, dw = (dz @ s["w"].float()).bfloat16(), (dz.T @ s["x"].float()).bfloat16()
    return dx, dw, (dz.sum(0) if s["b"] is not None else None)


def _offsets(c: dict):
    """[n, n]: the relative position (row major in what lies between two tokens of a window) of query i and key j."""
    h, w = c["high"], c["wide"]
    at = torch.arange(h * w, device=DEVICE)
    y, x = torch.div(at, w, rounding_mode="floor"), at % w
    return (y[:, None] - y + h - 1) * (2 * w - 1) + (x[:, None] - x + w - 1)


def _index(s):
    """[n, n]: the bucket of query i and key j."""
    at = _offsets(s["case"])
    return at if s["buckets"] is None else s["buckets"].long()[at]


def _plain_probs(s):
    """(q, k, v [windows, heads, n, d], probabilities, log2 of the sums of exponentials, buckets), fp32."""
    c = s["case"]
    n, heads, d = c["high"] * c["wide"], c["heads"], c["head_dim"]
    q, k, v = s["qkv"].float().view(-1, n, 3, heads, d).permute(2, 0, 3, 1, 4)
    index = _index(s)
    bias = s["table"].float().T[:, index]
    a = (q @ k.transpose(-1, -2)) * (1 / math.sqrt(d))
    a += torch.where(bias <= HIDDEN, -math.inf, bias)
    most = a.amax(-1, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    a = a.sub_(most).exp_()
    total = a.sum(-1, keepdim=True)
    # a query that sees nothing: zeros, and +inf so that exp(score - lse) is zero there too
    lse = torch.where(total > 0, (most + total.log()) * LOG2E, math.inf).squeeze(-1)
    a /= torch.where(total > 0, total, 1.0)
    return q, k, v, a, lse, index


def _together(x):
    """[windows, heads, n, d] -> [windows * n, heads * d]."""
    return x.permute(0, 2, 1, 3).flatten(2).flatten(0, 1)


def _plain_attn(s):
    _, _, v, p, lse, _ = _plain_probs(s)
    return _together(p @ v), lse


def _plain_attn_grad(s):
    c = s["case"]
    q, k, v, p, _, index = _plain_probs(s)
    d_o = s["d_o"].float().view(c["windows"], -1, c["heads"], c["head_dim"]).transpose(1, 2)
    dv = p.transpose(-1, -2) @ d_o
    ds = d_o @ v.transpose(-1, -2)
    ds -= (p * ds).sum(-1, keepdim=True)
    ds *= p
    scale = 1 / math.sqrt(c["head_dim"])
    dq, dk = scale * (ds @ k), scale * (ds.transpose(-1, -2) @ q)
    dqkv = torch.cat([_together(t) for t in (dq, dk, dv)], 1).bfloat16()
    sums = ds.double().sum(0).flatten(1) if c["windows"] * c["heads"] < 64 else ds.sum(0).double().flatten(1)
    dtable = torch.zeros((s["table"].shape[0], c["heads"]), dtype=torch.float64, device=DEVICE)
    dtable.index_add_(0, index.reshape(-1), sums.T)
    return dqkv, dtable.float()


def run(state: dict):
    s, c = state, state["case"]
    if own:
        if c["kind"].startswith("ln"):
            from aeris_gb_b200.ops import layer_norm as LN
            if c["kind"] == "ln":
                return LN.layer_norm_fwd(s["x"], s["w"], s["b"], eps=EPS)
            dx, dw, db = LN.layer_norm_bwd(s["dy"], s["x"], s["stats"], s["w"], bias=s["b"] is not None)
            return dx if s["w"] is None else (dx, dw, db)
        if c["kind"].startswith("lin"):
            from aeris_gb_b200.ops import linear as LI
            if c["kind"] == "lin":
                y, z = LI.linear_fwd(s["x"], s["w"], s["b"], act=c["act"], resid=s["resid"], keep=c["keep"])
                return (y, z) if c["keep"] else y
            return LI.linear_bwd(s["dy"], s["x"], s["w"], s["z"], act=c["act"], bias=s["b"] is not None)
        from aeris_gb_b200.ops import position_bias as PB
        shape = (c["windows"], (c["high"], c["wide"]), c["heads"], c["head_dim"])
        if c["kind"] == "attn":
            return PB.biased_attn_fwd(s["qkv"], *shape, s["table"], s["buckets"])
        return PB.biased_attn_bwd(s["d_o"], s["qkv"], s["o"], s["lse"], *shape, s["table"], s["buckets"])
    if c["kind"] == "ln":
        return _plain_ln(s)
    if c["kind"] == "ln-grad":
        return _plain_ln_grad(s)
    if c["kind"] == "lin":
        return _plain_lin(s)
    if c["kind"] == "lin-grad":
        return _plain_lin_grad(s)
    if c["kind"] == "attn":
        o, lse = _plain_attn(s)
        return o.bfloat16(), lse
    return _plain_attn_grad(s)


# ------------------------------------------------------------------------------------------------------------ floors
def work(case: dict) -> dict:
    c = case
    grad = c["kind"].endswith("grad")
    if c["kind"].startswith("ln"):
        size, n = (2 if c["dtype"] == "bfloat16" else 4), c["rows"] * c["cols"]
        side = 2 * c["cols"] * size * c["affine"] if not grad else c["cols"] * (size + 8) * c["affine"]
        return {"bytes": n * size * (3 if grad else 2) + 8 * c["rows"] + side, "flops": n * (12 if grad else 8)}
    if c["kind"].startswith("lin"):
        x, w, y = c["rows"] * c["inner"], c["inner"] * c["cols"], c["rows"] * c["cols"]
        if grad:
            # x, w and the gradient of y read, those of x and w written; the values before the activation read
            return {"bytes": 2 * (2 * x + 2 * w + y * (1 + (c["act"] != "none"))) + 4 * c["cols"] * c["bias"],
                    "flops": 4 * c["rows"] * w + 8 * y}
        return {"bytes": 2 * (x + w + y * (1 + c["resid"] + c["keep"])) + 4 * c["cols"] * c["bias"], "flops": 2 * c["rows"] * w + 8 * y}
    n, h, w = c["high"] * c["wide"], c["high"], c["wide"]
    t, inner, pairs = c["windows"] * n, c["heads"] * c["head_dim"], c["windows"] * c["heads"] * n * n
    table = 4 * (2 * h - 1) * (2 * w - 1) * c["heads"]
    if grad:      # qkv, o, its gradient and lse read, the gradient of qkv written; five products
        return {"bytes": 2 * t * 8 * inner + 4 * t * c["heads"] + 2 * table, "flops": pairs * (10 * c["head_dim"] + 10)}
    return {"bytes": 2 * t * 4 * inner + 4 * t * c["heads"] + table, "flops": pairs * (4 * c["head_dim"] + 6)}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _exact_ln(s):
    x = s["x"].double()
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    std = (var + EPS).sqrt()
    xhat = (x - mean) / std
    w = 1.0 if s["w"] is None else s["w"].double()
    if s["case"]["kind"] == "ln":
        return xhat * w + (0.0 if s["b"] is None else s["b"].double()), torch.cat([mean, 1 / std], 1)
    dy = s["dy"].double()
    g = dy * w
    # the gradient's parts along the row's constant and along xhat drop out
    n = x.shape[1]
    dx = (g - g.sum(1, keepdim=True) / n - xhat * ((g * xhat).sum(1, keepdim=True) / n)) / std
    return dx if s["w"] is None else (dx, torch.einsum("rc,rc->c", dy, xhat), dy.sum(0))


def _exact_lin(s):
    c = s["case"]
    if c["kind"] == "lin":
        z = torch.matmul(s["x"].double(), s["w"].double().T)
        if s["b"] is not None:
            z += s["b"].double()
    else:
        z = s["z"].double() if s["z"] is not None else None
    if c["act"] == "gelu":
        tail = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        f, df = z * tail, tail + z * (-z * z / 2).exp() / math.sqrt(2 * math.pi)
    elif c["act"] == "gelu_tanh":
        # (1 + tanh u) / 2 = sigmoid(2 u)
        u2 = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        p = torch.sigmoid(u2)
        f, df = z * p, p + z * p * (1 - p) * (2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2))
    elif c["act"] == "silu":
        p = torch.sigmoid(z)
        f, df = z * p, p + z * p * (1 - p)
    elif c["act"] == "relu":
        df = (z > 0).double()
        f = z * df
    else:
        f, df = z, None
    if c["kind"] == "lin":
        y = f if s["resid"] is None else f + s["resid"].double()
        return (y, z) if c["keep"] else y
    dz = s["dy"].double() if df is None else s["dy"].double() * df
    return (torch.matmul(dz, s["w"].double()), torch.matmul(s["x"].double().T, dz).T,
            torch.einsum("rc->c", dz) if s["b"] is not None else None)


def _exact_attn(s):
    c = s["case"]
    h, w, n, heads, d = c["high"], c["wide"], c["high"] * c["wide"], c["heads"], c["head_dim"]
    y, x = torch.meshgrid(torch.arange(h, device=DEVICE), torch.arange(w, device=DEVICE), indexing="ij")
    y, x = y.flatten(), x.flatten()
    at = (y.unsqueeze(1) - y.unsqueeze(0) + (h - 1)) * (2 * w - 1) + x.unsqueeze(1) - x.unsqueeze(0) + (w - 1)
    if s["buckets"] is not None:
        at = s["buckets"].to(torch.int64)[at]
    bias = s["table"].double()[at].permute(2, 0, 1)
    bias = bias.masked_fill(bias <= HIDDEN, -math.inf)
    grad = c["kind"] == "attn-grad"
    dtable = torch.zeros((s["table"].shape[0], heads), dtype=torch.float64, device=DEVICE)
    outs, lses = [], []
    step = max(1, int(2e8 // (heads * n * n)))
    for a in range(0, c["windows"], step):
        b = min(c["windows"], a + step)
        q, k, v = (t.squeeze(2) for t in s["qkv"][a * n:b * n].double().view(b - a, n, 3, heads, d).split(1, 2))
        score = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(d) + bias
        lse = torch.logsumexp(score, -1)
        lse = torch.where(lse == -math.inf, math.inf, lse)
        p = (score - lse.unsqueeze(-1)).exp()
        if not grad:
            outs.append(torch.einsum("bhij,bjhd->bihd", p, v).reshape(-1, heads * d))
            lses.append(lse / math.log(2.0))
            continue
        d_o = s["d_o"][a * n:b * n].double().view(b - a, n, heads, d)
        dp = torch.einsum("bihd,bjhd->bhij", d_o, v)
        ds = p * (dp - torch.einsum("bhij,bhij->bhi", p, dp).unsqueeze(-1))
        parts = [torch.einsum("bhij,bjhd->bihd", ds, k) / math.sqrt(d), torch.einsum("bhij,bihd->bjhd", ds, q) / math.sqrt(d),
                 torch.einsum("bhij,bihd->bjhd", p, d_o)]
        outs.append(torch.stack(parts, 2).reshape(-1, 3 * heads * d))
        dtable.index_add_(0, at.flatten(), ds.sum(0).flatten(1).T)
    return (torch.cat(outs), dtable) if grad else (torch.cat(outs), torch.cat(lses))


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return (_exact_ln if case["kind"].startswith("ln") else _exact_lin if case["kind"].startswith("lin") else _exact_attn)(s)
