"""Workloads of the operators that train a model on orthogonalised updates: the norms of queries and keys by head with the
position rotation in the same pass (forward and backward), the orthogonalisation of a batch of matrices, and a whole
optimizer step of the matrices of a flat parameter buffer (momentum, orthogonalisation, decay, weights, running average).

    listed()            the fixed cases
    draw(rng)           one more case from the ranges the fixed ones stand for
    prepare(case, seed) inputs on the GPU
    run(state)          one pass, in the operators' plain form or, where ``own`` is set, through the framework's entry points
    work(case)          bytes and floating-point operations that one pass cannot do without
    exact(case, seed)   what ``run`` returns, computed in 64 bits

Kinds of case: ``norm`` (queries and keys normed and rotated), ``norm-grad`` (its gradients), ``ortho`` (a batch of matrices
orthogonalised) and ``step`` (one optimizer step of ``layers`` blocks' matrices).
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
# p(x) = A x + B x^3 + C x^5, applied to the singular values once a step
A, B, C = 3.4445, -4.7750, 2.0315
STEPS = 5
LR, BETA, DECAY, SCALE, EMA_BETA, MAX_NORM = 2e-4, 0.95, 0.2, 0.2, 0.999, 20.0


# ------------------------------------------------------------------------------------------------------------ cases
def _norm(kind: str, rows: int, heads: int, kv_heads: int, head_dim: int, rotated: int, table: int, explicit: bool = False,
          fused: bool = True, dtype: str = "bfloat16") -> dict:
    """``rotated``: channels of a head that are rotated (0: none); ``table``: positions with an angle; ``explicit``: a
    position for each row (else row r is at r mod table); ``fused``: q and k are sections of one [rows, qkv] matrix."""
    return dict(kind=kind, rows=rows, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rotated=rotated, table=table,
                explicit=explicit, fused=fused, dtype=dtype)


def _ortho(count: int, rows: int, cols: int, dtype: str = "float32") -> dict:
    return dict(kind="ortho", count=count, rows=rows, cols=cols, dtype=dtype)


def _step(layers: int, dim: int, inner: int, mlp: int, ema: bool = True) -> dict:
    """Blocks of width ``dim`` with heads of ``inner`` channels in all and a gated MLP of ``mlp``."""
    return dict(kind="step", layers=layers, dim=dim, inner=inner, mlp=mlp, ema=ema)


def listed() -> list[dict]:
    cases = {
        # one token of the flagship's 24 heads of 64 at a position of its own: nothing but latency
        "norm-one-token": _norm("norm", 1, 24, 24, 64, 64, 900, explicit=True),
        # one 30 x 30 window of the flagship, out of the projection's [rows, q | k | v]
        "norm-window": _norm("norm", 900, 24, 24, 64, 64, 900),
        # odd sizes: shared key heads, a width that is no power of two, half of it rotated, fp32, tensors of their own
        "norm-odd": _norm("norm", 12345, 10, 2, 72, 40, 257, explicit=True, fused=False, dtype="float32"),
        # a chunk of 72 windows of the flagship, what a block's forward pass works on at a time
        "norm-chunk": _norm("norm", 64800, 24, 24, 64, 64, 900),
        # the gradients of a toy model: 16 windows of 8 x 8 tokens, two heads of 32
        "norm-grad-toy": _norm("norm-grad", 1024, 2, 2, 32, 32, 64),
        # and of the flagship's chunk
        "norm-grad-chunk": _norm("norm-grad", 64800, 24, 24, 64, 64, 900),
        # and of the wide model's 40 heads of 128, 32 windows
        "norm-grad-wide": _norm("norm-grad", 28800, 40, 40, 128, 128, 900),
        # a toy model's matrices: the smallest calls
        "ortho-toy": _ortho(8, 64, 64),
        # odd, upright matrices
        "ortho-odd": _ortho(10, 1001, 333),
        # one MLP matrix of the wide model, from bf16
        "ortho-wide": _ortho(1, 5120, 13696, "bfloat16"),
        # a small model's whole step
        "step-small": _step(6, 384, 384, 1024),
        # four blocks of the flagship
        "step-flagship": _step(4, 1536, 1536, 4096),
    }
    return [{"name": name, **c} for name, c in cases.items()]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm-grad", "ortho", "step"])
    if kind.startswith("norm"):
        kv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24, 40])
        heads = kv * rng.choice([1, 1, 1, 2, 4]) if kv <= 12 else kv
        d = rng.choice([8, 16, 24, 32, 40, 48, 64, 64, 72, 80, 96, 104, 128, 128, 192, 256, 20, 36, 100])
        most = 40 * 2 * 128 * 28800 // ((heads + kv) * d)
        rows = _log_int(rng, 1, min(65536, most))
        rotated = rng.choice([0, d, d, d, d // 4 * 2])
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        if dtype == "float32":
            rows = max(1, rows // 2)
        return _norm(kind, rows, heads, kv, d, rotated, _log_int(rng, 1, 4096), rng.random() < 0.5, rng.random() < 0.7, dtype)
    if kind == "ortho":
        rows, cols = _log_int(rng, 1, 5120), _log_int(rng, 1, 13696)
        if rng.random() < 0.5:
            rows, cols = cols, rows
        d, k = min(rows, cols), max(rows, cols)
        most = 60 * 5120 ** 3 / (d * d * (4 * k + 2 * d) * 5) + 1
        count = _log_int(rng, 1, max(1, min(48, int(most), int(3e8 / (d * k)))))
        return _ortho(count, rows, cols, rng.choice(["float32", "float32", "bfloat16"]))
    dim = rng.choice([64, 96, 128, 200, 256, 384, 500, 512, 768, 896, 1024, 1536])
    inner = rng.choice([dim, dim, dim // 2])
    mlp = _log_int(rng, dim, 4 * dim)
    layers = _log_int(rng, 1, 24 if dim <= 512 else 6)
    return _step(layers, dim, inner, mlp, rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------------------ inputs
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(1000003 * seed + 17)


def _matrices(c: dict) -> list[tuple[int, int, int]]:
    """(rows, cols, how many) of a step's groups: q, k, v sections; wo; gate and up halves of w1; w2."""
    n, dim, inner, mlp = (c[k] for k in ("layers", "dim", "inner", "mlp"))
    return [(inner, dim, 3 * n), (dim, inner, n), (mlp, dim, 2 * n), (dim, mlp, n)]


def _gradient(g: torch.Generator, count: int, rows: int, cols: int) -> torch.Tensor:
    """Gradient-like matrices: a few strong directions whose strength falls off, and the noise of a batch. fp32."""
    r = min(rows, cols, 64)
    strength = torch.arange(1, r + 1, device=DEVICE, dtype=torch.float32).rsqrt()
    u = torch.randn((count, rows, r), generator=g, device=DEVICE) * strength
    v = torch.randn((count, r, cols), generator=g, device=DEVICE)
    signal = torch.bmm(u, v)
    signal *= 1.0 / signal.pow(2).mean().sqrt().clamp_min(1e-20)
    signal += 0.5 * torch.randn((count, rows, cols), generator=g, device=DEVICE)
    return signal.mul_(1e-3)


def prepare(case: dict, seed: int) -> dict:
    c, g = case, _generator(seed)
    s = {"case": c}
    if c["kind"] in ("norm", "norm-grad"):
        rows, H, Hk, d, dt = c["rows"], c["heads"], c["kv_heads"], c["head_dim"], getattr(torch, c["dtype"])

        def pair(scale):
            if not c["fused"]:
                return tuple((scale * torch.randn((rows, n, d), generator=g, device=DEVICE)).to(dt) for n in (H, Hk))
            x = (scale * torch.randn((rows, (H + 2 * Hk) * d), generator=g, device=DEVICE)).to(dt)
            return x[:, :H * d].view(rows, H, d), x[:, H * d:(H + Hk) * d].view(rows, Hk, d)

        s["q"], s["k"] = pair(1.5)
        # channels of unlike strength, as a trained projection has them
        s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(d, generator=g, device=DEVICE)).to(dt) for _ in range(2))
        s["cos"] = s["sin"] = s["positions"] = None
        if c["rotated"]:
            half = c["rotated"] // 2
            theta = 10000.0 ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
            ang = torch.outer(torch.arange(c["table"], device=DEVICE, dtype=torch.float64), theta)
            s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
            if c["explicit"]:
                s["positions"] = torch.randint(0, c["table"], (rows,), generator=g, device=DEVICE, dtype=torch.int32)
        if c["kind"] == "norm-grad":
            s["dq"], s["dk"] = pair(0.01)
    elif c["kind"] == "ortho":
        s["x"] = _gradient(g, c["count"], c["rows"], c["cols"]).to(getattr(torch, c["dtype"]))
    else:
        groups, total = [], 0
        for rows, cols, n in _matrices(c):
            at = []
            for _ in range(n):
                at.append(total)
                total += (rows * cols + 15) // 16 * 16
            groups.append((rows, cols, at))
        grad, mom = torch.zeros(total, device=DEVICE), torch.zeros(total, device=DEVICE)
        for rows, cols, at in groups:
            new, old = _gradient(g, len(at), rows, cols), _gradient(g, len(at), rows, cols)
            for i, o in enumerate(at):
                grad[o:o + rows * cols] = new[i].reshape(-1)
                mom[o:o + rows * cols] = old[i].reshape(-1)
        s["groups"] = [(rows, cols, torch.tensor(at, dtype=torch.int64, device=DEVICE)) for rows, cols, at in groups]
        s["at"] = [at for _, _, at in groups]
        s["grad"], s["momentum"] = grad, mom
        s["master"] = 0.02 * torch.randn(total, generator=g, device=DEVICE)
        s["weights"] = s["master"].bfloat16()
        s["ema"] = s["master"] + 1e-4 * torch.randn(total, generator=g, device=DEVICE) if c["ema"] else None
        s["norm_sq"] = (16.0 * MAX_NORM ** 2) * torch.ones(1, dtype=torch.float64, device=DEVICE)    # clipped to a quarter
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _angles(s, rows: int):
    """cos and sin of every row, [rows, 1, rotated / 2]."""
    if s["positions"] is not None:
        at = s["positions"].long()
    else:
        at = torch.arange(rows, device=DEVICE) % s["cos"].shape[0]
    return s["cos"][at].unsqueeze(1), s["sin"][at].unsqueeze(1)


def _rotate(y, s, sign: float):
    if s["cos"] is None:
        return y
    cos, sin = _angles(s, y.shape[0])
    n = 2 * cos.shape[-1]
    a, b, sin = y[..., 0:n:2], y[..., 1:n:2], sign * sin
    turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, y[..., n:]], -1) if n < y.shape[-1] else turned


def _plain_norm(x, w, s):
    xf = x.float()
    y = xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS) * w.float()
    return _rotate(y, s, 1.0).to(x.dtype)


def _plain_norm_grad(dy, x, w, s):
    xf = x.float()
    r = torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS)
    xhat, dz = xf * r, _rotate(dy.float(), s, -1.0)
    dw = (dz * xhat).sum((0, 1))
    g = dz * w.float()
    return (r * (g - xhat * (g * xhat).mean(-1, keepdim=True))).to(x.dtype), dw


def _plain_ortho(x):
    """[count, rows, cols] fp32 -> fp32."""
    t = x.shape[1] > x.shape[2]
    y = x.transpose(1, 2) if t else x
    y = y / y.double().square().sum((1, 2), keepdim=True).sqrt().float().clamp_min(1e-7)
    for _ in range(STEPS):
        m = torch.bmm(y, y.transpose(1, 2))
        y = A * y + torch.bmm(B * m + C * torch.bmm(m, m), y)
    return y.transpose(1, 2) if t else y


def _plain_step(s):
    clip = (MAX_NORM / (s["norm_sq"].sqrt() + 1e-6)).clamp(max=1.0).float()
    for (rows, cols, _), at in zip(s["groups"], s["at"]):
        n = rows * cols
        views = lambda t: torch.stack([t[o:o + n].view(rows, cols) for o in at])  # noqa: E731
        g = torch.nan_to_num(views(s["grad"]) * clip, nan=0.0, posinf=1e5, neginf=-1e5)
        m = BETA * views(s["momentum"]) + (1 - BETA) * g
        o = _plain_ortho(BETA * m + (1 - BETA) * g)
        p = views(s["master"]) * (1 - LR * DECAY) - LR * SCALE * math.sqrt(max(rows, cols)) * o
        for i, a in enumerate(at):
            s["momentum"][a:a + n] = m[i].reshape(-1)
            s["master"][a:a + n] = p[i].reshape(-1)
            s["weights"][a:a + n] = p[i].reshape(-1).bfloat16()
            if s["ema"] is not None:
                s["ema"][a:a + n].sub_(p[i].reshape(-1)).mul_(EMA_BETA).add_(p[i].reshape(-1))


def _step_outputs(s):
    return {k: s[k] for k in ("master", "momentum", "weights", "ema") if s[k] is not None}


def run(state: dict):
    s, kind = state, state["case"]["kind"]
    if own:
        if kind.startswith("norm"):
            from aeris_gb_b200.ops import qk_norm as QN
        else:
            from aeris_gb_b200.ops import orthogonalise as OR
        if kind == "norm":
            return QN.qk_norm_fwd(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], eps=EPS, positions=s["positions"])
        if kind == "norm-grad":
            return QN.qk_norm_bwd(s["dq"], s["dk"], s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], eps=EPS,
                                  positions=s["positions"])
        if kind == "ortho":
            return OR.orthogonalise(s["x"], steps=STEPS)
        OR.orthogonal_step(s["master"], s["grad"], s["momentum"], s["weights"], s["ema"], s["norm_sq"], groups=s["groups"],
                           lr=LR, beta=BETA, nesterov=True, weight_decay=DECAY, scale=SCALE, grad_scale=1.0,
                           max_norm=MAX_NORM, ema_beta=EMA_BETA, steps=STEPS, zero_grad=False)
        return _step_outputs(s)
    if kind == "norm":
        return _plain_norm(s["q"], s["wq"], s), _plain_norm(s["k"], s["wk"], s)
    if kind == "norm-grad":
        dq, dwq = _plain_norm_grad(s["dq"], s["q"], s["wq"], s)
        dk, dwk = _plain_norm_grad(s["dk"], s["k"], s["wk"], s)
        return dq, dk, dwq, dwk
    if kind == "ortho":
        return _plain_ortho(s["x"].float()).bfloat16().contiguous()
    _plain_step(s)
    return _step_outputs(s)


# ------------------------------------------------------------------------------------------------------------ floors
def _ortho_flops(rows: int, cols: int) -> float:
    """Of one matrix, symmetric products counted at half. A step by itself takes (in units of d^3, r = longer / shorter side)
    r for the Gram matrix, 1 for its square and 2 r for the update: 3 r + 1. Three steps, or two, on the Gram matrix alone
    with one update at their end take 3 r + 9, or 3 r + 5. The cheaper of the two ways."""
    d, k = min(rows, cols), max(rows, cols)
    r = k / d
    return min(STEPS * (3 * r + 1), 6 * r + 14) * d ** 3


def work(case: dict) -> dict:
    c = case
    if c["kind"].startswith("norm"):
        size = 2 if c["dtype"] == "bfloat16" else 4
        n = c["rows"] * (c["heads"] + c["kv_heads"]) * c["head_dim"]
        grad = c["kind"] == "norm-grad"
        side = c["table"] * c["rotated"] * 4 + 2 * c["head_dim"] * (size + 4 * grad) + (4 * c["rows"] if c["explicit"] else 0)
        return {"bytes": n * size * (3 if grad else 2) + side, "flops": n * (16 if grad else 8)}
    if c["kind"] == "ortho":
        n = c["count"] * c["rows"] * c["cols"]
        return {"bytes": n * (2 + (2 if c["dtype"] == "bfloat16" else 4)),
                "flops": c["count"] * _ortho_flops(c["rows"], c["cols"])}
    groups = _matrices(c)
    n = sum(r * k * m for r, k, m in groups)
    # gradient read; momentum and weights read and written, bf16 weights written, running average read and written
    return {"bytes": n * (4 + 8 + 8 + 2 + (8 if c["ema"] else 0)), "flops": sum(m * _ortho_flops(r, k) for r, k, m in groups)}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _exact_turn(s, rows: int):
    """The rotation of every row as complex numbers [rows, 1, rotated / 2], from the angles' table that the call is given."""
    at = s["positions"].long() if s["positions"] is not None else torch.remainder(torch.arange(rows, device=DEVICE),
                                                                                 s["cos"].shape[0])
    return torch.complex(s["cos"].double(), s["sin"].double())[at][:, None, :]


def _exact_rotated(y, s, back: bool):
    if s["cos"] is None:
        return y
    z = _exact_turn(s, y.shape[0])
    n = 2 * z.shape[-1]
    head = torch.view_as_complex(y[..., :n].unflatten(-1, (n // 2, 2)).contiguous())
    head = torch.view_as_real(head * (z.conj() if back else z)).flatten(-2)
    return torch.cat([head, y[..., n:]], -1)


def _exact_ortho(x):
    """Through the eigenvalues of the smaller Gram matrix nothing would be gained: the iteration itself, in 64 bits."""
    x = x.double()
    if x.shape[0] > x.shape[1]:
        return _exact_ortho(x.T).T
    x = x / max(torch.linalg.matrix_norm(x).item(), 1e-7)
    one = torch.eye(x.shape[0], dtype=torch.float64, device=DEVICE)
    for _ in range(STEPS):
        gram = x @ x.T
        x = (A * one + gram @ (B * one + C * gram)) @ x
    return x


def exact(case: dict, seed: int):
    s, kind = prepare(case, seed), case["kind"]
    if kind.startswith("norm"):
        out, sums = [], []
        for x, w, dy in ((s["q"], s["wq"], s.get("dq")), (s["k"], s["wk"], s.get("dk"))):
            x, w = x.double(), w.double()
            rms = ((x * x).mean(-1, keepdim=True) + EPS).sqrt()
            if kind == "norm":
                out.append(_exact_rotated(x / rms * w, s, False))
                continue
            dz = _exact_rotated(dy.double(), s, True)
            sums.append((dz * x / rms).sum((0, 1)))
            dx = dz * w / rms
            out.append(dx - x * (dx * x).mean(-1, keepdim=True) / rms ** 2)
        return tuple(out + sums)
    if kind == "ortho":
        return torch.stack([_exact_ortho(x) for x in s["x"]])
    clip = min(1.0, MAX_NORM / (math.sqrt(s["norm_sq"].item()) + 1e-6))
    new = {k: s[k].double() for k in ("master", "momentum", "ema") if s[k] is not None}
    new["weights"] = s["weights"].double()
    for (rows, cols, _), at in zip(s["groups"], s["at"]):
        for o in at:
            sl = slice(o, o + rows * cols)
            g = s["grad"][sl].double() * clip
            m = BETA * s["momentum"][sl].double() + (1 - BETA) * g
            u = _exact_ortho((BETA * m + (1 - BETA) * g).view(rows, cols)).reshape(-1)
            p = (1 - LR * DECAY) * s["master"][sl].double() - LR * SCALE * math.sqrt(max(rows, cols)) * u
            new["momentum"][sl], new["master"][sl], new["weights"][sl] = m, p, p
            if s["ema"] is not None:
                new["ema"][sl] = p + EMA_BETA * (s["ema"][sl].double() - p)
    return {k: new[k] for k in ("master", "momentum", "weights", "ema") if k in new}
