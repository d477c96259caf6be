"""Norms of queries and keys with the rotation against their formulas in 64 bits.

Tolerances: a result in type t is rounded once, by half a step eps(t) / 2 of its value. Before that everything is fp32: a value
is a handful of operations (16 roundings of 2^-24 are allowed for, a reciprocal root of 2 steps among them) on terms whose sizes
are added up instead of the result, which a cancellation can leave small; sums over d channels add (log2 d + 8) roundings of
the terms' absolute sum. Sums over rows: as many roundings as there are terms, of their absolute sum.
"""
import math

import pytest
import torch

from aeris_gb_b200.ops import lib as _l
from aeris_gb_b200.ops import qk_norm as QN

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def turn(y, cos, sin, at, back=False):
    if cos is None:
        return y
    n = 2 * cos.shape[1]
    c, s = cos.double()[at][:, None], sin.double()[at][:, None] * (-1 if back else 1)
    e, o = y[..., 0:n:2], y[..., 1:n:2]
    return torch.cat([torch.stack([e * c - o * s, o * c + e * s], -1).flatten(-2), y[..., n:]], -1)


def pair_size(y, n):
    """Sizes of both terms of a rotated pair, summed."""
    a = y.abs()
    p = (a[..., 0:n:2] + a[..., 1:n:2]).repeat_interleave(2, -1)
    return torch.cat([p, a[..., n:]], -1)


def formula(x, w, cos, sin, at, eps, dy=None):
    """(y, size of its terms) and, with ``dy``, (dx, size, dw, size), in 64 bits."""
    x, w = x.double(), w.double()
    n = 0 if cos is None else 2 * cos.shape[1]
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    z = x * r * w
    if dy is None:
        return turn(z, cos, sin, at), pair_size(z, n)
    dz, size = turn(dy.double(), cos, sin, at, True), pair_size(dy.double(), n)
    xhat, g = x * r, dz * w
    dx = r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    mean = (size * w.abs() * xhat.abs()).mean(-1, keepdim=True)
    dx_size = r * (size * w.abs() + xhat.abs() * mean * (math.log2(x.shape[-1]) + 8))
    return dx, dx_size, (dz * xhat).sum((0, 1)), (size * xhat.abs()).sum((0, 1))


def close(got, want, size, dt, roundings=16):
    bound = half_step(dt) * (want.abs() + roundings * U * size) + roundings * U * size + 1e-30
    assert bool(((got.double() - want).abs() <= bound).all()), ((got.double() - want).abs() / bound).max().item()


def make(rows, H, Hk, d, rot, L, dt, wdt=None, explicit=None, layout="fused", seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731

    def pair():
        if layout == "fused":
            x = rnd(rows, (H + 2 * Hk) * d).to(dt)
            return x[:, :H * d].unflatten(1, (H, d)), x[:, H * d:(H + Hk) * d].unflatten(1, (Hk, d))
        if layout == "heads first":
            return tuple(rnd(n, rows, d).to(dt).transpose(0, 1) for n in (H, Hk))
        if layout == "odd start":
            return tuple(rnd(rows, n * d + 3).to(dt)[:, 1:1 + n * d].unflatten(1, (n, d)) for n in (H, Hk))
        return tuple(rnd(rows, n, d).to(dt) for n in (H, Hk))

    q, k = pair()
    dq, dk = pair()
    wq, wk = (1 + 0.3 * rnd(d)).to(wdt or dt), (1 + 0.3 * rnd(d)).to(wdt or dt)
    cos = sin = pos = None
    at = None
    if rot:
        ang = 20 * rnd(L, rot // 2)
        cos, sin = ang.cos(), ang.sin()
        at = torch.arange(rows, device=DEV) % L
        if explicit:
            at = torch.randint(0, L, (rows,), generator=g, device=DEV)
            pos = at.to(explicit)
    return q, k, dq, dk, wq, wk, cos, sin, pos, at


CASES = [  # rows, heads, kv heads, d, rot, L, type, weights, positions, layout
    (1, 1, 1, 2, 2, 1, torch.float32, None, None, "own"),
    (1, 24, 24, 64, 64, 900, torch.bfloat16, None, torch.int32, "fused"),
    (1, 40, 40, 128, 128, 7, torch.bfloat16, None, torch.int64, "fused"),
    (3, 5, 1, 8, 8, 2, torch.bfloat16, None, None, "own"),
    (7, 3, 3, 16, 0, 1, torch.bfloat16, torch.float32, None, "fused"),
    (65, 6, 2, 24, 24, 64, torch.bfloat16, None, None, "heads first"),
    (257, 8, 8, 32, 16, 100, torch.float32, None, torch.int64, "fused"),
    (900, 4, 4, 64, 64, 900, torch.bfloat16, None, None, "fused"),
    (333, 7, 7, 72, 40, 31, torch.bfloat16, torch.float32, torch.int32, "own"),
    (129, 3, 1, 80, 78, 50, torch.bfloat16, None, None, "fused"),          # a rotation that ends inside a vector
    (200, 2, 2, 96, 96, 200, torch.float32, torch.bfloat16, None, "own"),
    (1000, 3, 3, 128, 128, 1000, torch.bfloat16, None, None, "odd start"),
    (50, 33, 11, 36, 36, 9, torch.bfloat16, None, None, "own"),
    (41, 2, 1, 100, 50, 41, torch.float32, None, torch.int32, "odd start"),
    (77, 3, 2, 192, 64, 5, torch.bfloat16, None, None, "own"),
    (19, 2, 2, 256, 256, 19, torch.bfloat16, None, torch.int32, "heads first"),
    (11, 2, 2, 254, 254, 11, torch.float32, None, None, "own"),
    (4099, 2, 2, 32, 32, 64, torch.bfloat16, None, None, "fused"),
    # widths of whole fours, with every kind of rotation
    (257, 5, 3, 20, 10, 33, torch.bfloat16, None, torch.int32, "own"),
    (300, 9, 2, 36, 18, 100, torch.bfloat16, torch.float32, None, "fused"),
    (101, 4, 4, 100, 50, 101, torch.bfloat16, None, None, "own"),
    (64, 3, 3, 100, 100, 64, torch.float32, None, torch.int64, "heads first"),
    (90, 7, 1, 12, 12, 9, torch.float32, None, None, "own"),
    (33, 2, 2, 4, 4, 33, torch.bfloat16, None, None, "own"),
    (120, 6, 6, 128, 60, 40, torch.bfloat16, None, None, "fused"),
    (77, 2, 2, 252, 130, 7, torch.bfloat16, None, None, "own"),
    (59, 3, 2, 256, 256, 59, torch.float32, None, None, "own"),
    # groups of three, five, six, nine and ten lanes
    (210, 11, 4, 24, 24, 70, torch.bfloat16, None, None, "own"),
    (211, 13, 5, 40, 20, 71, torch.float32, None, torch.int32, "fused"),
    (212, 6, 2, 48, 48, 72, torch.bfloat16, None, None, "fused"),
    (213, 4, 3, 72, 72, 73, torch.bfloat16, None, None, "own"),
    (214, 7, 2, 80, 80, 74, torch.float32, None, None, "heads first"),
    # steps that take heads of several rows, up to a row that is the last of them
    (1001, 1, 1, 8, 8, 100, torch.bfloat16, None, torch.int32, "own"),
    (1003, 2, 1, 64, 64, 1003, torch.bfloat16, None, None, "fused"),
    (2049, 3, 1, 24, 12, 50, torch.float32, None, torch.int64, "fused"),
    (515, 4, 1, 16, 16, 515, torch.bfloat16, None, None, "heads first"),
    (5, 1, 1, 2, 2, 5, torch.float32, None, None, "own"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_forward(case):
    q, k, _, _, wq, wk, cos, sin, pos, at = make(*case)
    yq, yk = QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6, positions=pos)
    for x, w, y in ((q, wq, yq), (k, wk, yk)):
        close(y, *formula(x, w, cos, sin, at, 1e-6), q.dtype)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_backward(case):
    q, k, dq, dk, wq, wk, cos, sin, pos, at = make(*case)
    gq, gk, gwq, gwk = QN.qk_norm_bwd(dq, dk, q, k, wq, wk, cos, sin, eps=1e-6, positions=pos)
    for x, w, dy, dx, dw in ((q, wq, dq, gq, gwq), (k, wk, dk, gk, gwk)):
        ex, size, ew, wsize = formula(x, w, cos, sin, at, 1e-6, dy)
        close(dx, ex, size, q.dtype)
        close(dw, ew, wsize, torch.float32, 16 + x.shape[0] * x.shape[1])


def test_backward_equals_differences():
    """Against differences of the formula itself: central, step h, error h^2 / 6 of the third derivative, far below 1e-6."""
    q, k, dq, dk, wq, wk, cos, sin, pos, at = make(5, 2, 1, 8, 8, 3, torch.float32)
    gq, _, gwq, _ = QN.qk_norm_bwd(dq, dk, q, k, wq, wk, cos, sin, eps=1e-2)
    loss = lambda x, w: (formula(x, w, cos, sin, at, 1e-2)[0] * dq.double()).sum()  # noqa: E731
    h = 1e-4
    x, w = q.double(), wq.double()
    for got, base, at_base in ((gq, x, lambda v: loss(v, w)), (gwq, w, lambda v: loss(x, v))):
        num = torch.empty_like(base)
        for i in range(base.numel()):
            e = torch.zeros(base.numel(), dtype=torch.float64, device=DEV)
            e[i] = h
            e = e.view(base.shape)
            num.view(-1)[i] = (at_base(base + e) - at_base(base - e)) / (2 * h)
        assert (got.double() - num).abs().max() <= 1e-5 * max(1.0, num.abs().max().item())


def test_rows_of_zeros_and_large_values():
    q, k, dq, dk, wq, wk, cos, sin, _, at = make(64, 2, 2, 64, 64, 64, torch.bfloat16)
    q, k = q.clone(), k.clone()
    q[3] = 0
    q[5] *= 2.0 ** 60                # its squares end at 2^120 x 64: inside fp32
    yq, _ = QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6)
    gq, *_ = QN.qk_norm_bwd(dq, dk, q, k, wq, wk, cos, sin, eps=1e-6)
    assert bool((yq[3] == 0).all()) and bool(yq.isfinite().all()) and bool(gq.isfinite().all())
    close(yq, *formula(q, wq, cos, sin, at, 1e-6), q.dtype)
    ex, size, *_ = formula(q, wq, cos, sin, at, 1e-6, dq)
    close(gq, ex, size, q.dtype)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_one_row_of_nan_stays_one_row(dt):
    q, k, dq, dk, wq, wk, cos, sin, _, _ = make(40, 3, 3, 32, 32, 40, dt)
    want = QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6)[0]
    q[7, 1, 5] = float("nan")
    got = QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6)[0]
    assert bool(got[7, 1].isnan().all())
    got[7, 1] = want[7, 1]
    assert torch.equal(got, want)


def same_or_close(got, want, size, dt, roundings=16):
    """:func:`close` where ``want`` is a number; elsewhere the same infinity, or no number in both."""
    ok = want.isfinite() & size.isfinite()
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[want.isinf()], want[want.isinf()])
    close(got[ok], want[ok], size[ok], dt, roundings)


@pytest.mark.parametrize("d,rot,dt", [(64, 32, torch.bfloat16), (64, 0, torch.bfloat16), (72, 40, torch.bfloat16), (36, 18, torch.bfloat16),
                                      (100, 50, torch.bfloat16), (80, 78, torch.bfloat16), (254, 100, torch.bfloat16),
                                      (64, 32, torch.float32), (36, 18, torch.float32), (20, 2, torch.float32), (30, 14, torch.float32)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_a_channel_that_is_not_turned_leaves_its_neighbour_alone(d, rot, dt, value):
    """Infinities and NaN in the weights, in q and in the results' gradient, in channels behind the turned ones."""
    rows = 9
    q, k, dq, dk, wq, wk, cos, sin, _, at = make(rows, 3, 2, d, rot, rows, dt, layout="own")
    for what in ("weight", "q", "dq"):
        for c in {rot, rot + 1, d - 1}:
            x, w, dy = q.clone(), wq.clone(), dq.clone()
            if what == "weight":
                w[c] = value
            else:
                (x if what == "q" else dy)[4, 1, c] = value
            y, _ = QN.qk_norm_fwd(x, k, w, wk, cos, sin, eps=1e-6)
            same_or_close(y, *formula(x, w, cos, sin, at, 1e-6), dt)
            if what == "q":                      # the root is zero or no number: nothing of this head's gradient is left
                continue
            dx, _, dw, _ = QN.qk_norm_bwd(dy, dk, x, k, w, wk, cos, sin, eps=1e-6)
            ex, size, ew, wsize = formula(x, w, cos, sin, at, 1e-6, dy)
            same_or_close(dx, ex, size, dt)
            same_or_close(dw, ew, wsize, torch.float32, 16 + 3 * rows)


@pytest.mark.parametrize("d", [64, 36])
def test_in_place_and_into_sections(d):
    """Results over the inputs, and into sections of one matrix whose rest is left as it was."""
    rows, H, Hk = 75, 4, 2
    q, k, dq, dk, wq, wk, cos, sin, _, _ = make(rows, H, Hk, d, d, 75, torch.bfloat16, layout="own")
    yq, yk = QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6)
    gq, gk, gwq, gwk = QN.qk_norm_bwd(dq, dk, q, k, wq, wk, cos, sin, eps=1e-6)
    whole = torch.full((rows + 2, (H + 2 * Hk) * d), 7.0, device=DEV, dtype=torch.bfloat16)
    sq = whole[1:-1, :H * d].unflatten(1, (H, d))
    sk = whole[1:-1, H * d:(H + Hk) * d].unflatten(1, (Hk, d))
    QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6, q_out=sq, k_out=sk)
    assert torch.equal(sq, yq) and torch.equal(sk, yk)
    assert bool((whole[:, (H + Hk) * d:] == 7).all()) and bool((whole[[0, -1]] == 7).all())
    dw = torch.full((2, d), 3.0, device=DEV)
    QN.qk_norm_bwd(dq, dk, q, k, wq, wk, cos, sin, eps=1e-6, dq_out=dq, dk_out=dk, dwq=dw[0], dwk=dw[1])
    assert torch.equal(dq, gq) and torch.equal(dk, gk)
    assert (dw[0] - 3 - gwq).abs().max() <= 4 * U * (3 + gwq.abs().max()) and (dw[1] - 3 - gwk).abs().max() <= 4 * U * (
        3 + gwk.abs().max())
    QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6, q_out=q, k_out=k)
    assert torch.equal(q, yq) and torch.equal(k, yk)


@pytest.mark.parametrize("heads,d,dt", [(5, 64, torch.bfloat16), (1, 24, torch.float32), (3, 100, torch.bfloat16), (5, 72, torch.float32)])
def test_without_eps(heads, d, dt):
    """Places of a step that hold no head have a root of zero, which must not reach the sums."""
    q, k, dq, dk, wq, wk, cos, sin, _, at = make(37, heads, heads, d, d, 37, dt)
    yq, _ = QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=0.0)
    close(yq, *formula(q, wq, cos, sin, at, 0.0), dt)
    gq, _, gwq, gwk = QN.qk_norm_bwd(dq, dk, q, k, wq, wk, cos, sin, eps=0.0)
    ex, size, ew, wsize = formula(q, wq, cos, sin, at, 0.0, dq)
    close(gq, ex, size, dt)
    close(gwq, ew, wsize, torch.float32, 16 + 37 * heads)
    assert bool(gwk.isfinite().all())


@pytest.mark.parametrize("rows,d", [(1, 16), (700, 64), (33, 250)])
def test_a_weight_that_q_and_k_share(rows, d):
    """One tensor for both gradients: the sum of both."""
    q, k, dq, dk, w, _, cos, sin, _, at = make(rows, 4, 2, d, d, rows, torch.bfloat16)
    dw = torch.full((d,), 3.0, device=DEV)
    QN.qk_norm_bwd(dq, dk, q, k, w, w, cos, sin, eps=1e-6, dwq=dw, dwk=dw)
    _, _, eq, size_q = formula(q, w, cos, sin, at, 1e-6, dq)
    _, _, ek, size_k = formula(k, w, cos, sin, at, 1e-6, dk)
    close(dw, 3 + eq + ek, 3 + size_q + size_k, torch.float32, 16 + 6 * rows)


def test_few_query_heads_beside_many_key_heads():
    q, k, dq, dk, wq, wk, cos, sin, _, at = make(50, 1, 2001, 8, 8, 50, torch.bfloat16, layout="own")
    yq, yk = QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6)
    gq, gk, gwq, gwk = QN.qk_norm_bwd(dq, dk, q, k, wq, wk, cos, sin, eps=1e-6)
    for x, w, dy, y, dx, dw in ((q, wq, dq, yq, gq, gwq), (k, wk, dk, yk, gk, gwk)):
        close(y, *formula(x, w, cos, sin, at, 1e-6), q.dtype)
        ex, size, ew, wsize = formula(x, w, cos, sin, at, 1e-6, dy)
        close(dx, ex, size, q.dtype)
        close(dw, ew, wsize, torch.float32, 16 + x.shape[0] * x.shape[1])


def test_no_rows():
    q, k, dq, dk, wq, wk, cos, sin, _, _ = make(0, 4, 2, 16, 16, 4, torch.bfloat16)
    before = _l.launch_count()
    yq, yk = QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6)
    gq, gk, gwq, gwk = QN.qk_norm_bwd(dq, dk, q, k, wq, wk, cos, sin, eps=1e-6)
    assert yq.shape == gq.shape == (0, 4, 16) and yk.shape == gk.shape == (0, 2, 16)
    assert bool((gwq == 0).all()) and bool((gwk == 0).all()) and _l.launch_count() == before


@pytest.mark.parametrize("bad", [-1, 5, 2 ** 31 - 1])
def test_position_outside_the_table_is_reported_and_its_row_left(bad):
    q, k, dq, dk, wq, wk, cos, sin, _, _ = make(9, 2, 2, 32, 32, 5, torch.bfloat16, layout="own")
    pos = torch.arange(9, device=DEV, dtype=torch.int32) % 5
    pos[4] = bad
    yq, yk = torch.full_like(q, 7), torch.full_like(k, 7)
    QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6, positions=pos, q_out=yq, k_out=yk)
    with pytest.raises(_l.KernelError, match="bounds"):
        _l.check_status()
    good = [i for i in range(9) if i != 4]
    want = QN.qk_norm_fwd(q[good], k[good], wq, wk, cos, sin, eps=1e-6, positions=pos[good])
    assert torch.equal(yq[good], want[0]) and torch.equal(yk[good], want[1]) and bool((yq[4] == 7).all())
    out = QN.qk_norm_bwd(dq, dk, q, k, wq, wk, cos, sin, eps=1e-6, positions=pos, dq_out=yq, dk_out=yk)
    with pytest.raises(_l.KernelError, match="bounds"):
        _l.check_status()
    want = QN.qk_norm_bwd(dq[good], dk[good], q[good], k[good], wq, wk, cos, sin, eps=1e-6, positions=pos[good])
    assert torch.equal(out[0][good], want[0]) and bool((yk[4] == 7).all())
    close(out[2], want[2].double(), (dq.abs().float().sum((0, 1)) * 8).double(), torch.float32)     # the row takes no part


def test_rows_beyond_32_bit_offsets():
    """Row 40,000 of a matrix whose rows are 120,000 elements apart lies behind 2^32 elements."""
    rows, H, d, pitch = 40001, 1, 64, 120000
    base = torch.empty(rows * pitch, dtype=torch.bfloat16, device=DEV)
    q = base.as_strided((rows, H, d), (pitch, d, 1))
    k = base.as_strided((rows, H, d), (pitch, d, 1), d)
    src = torch.randn(2, rows, H, d, device=DEV).bfloat16()
    q.copy_(src[0])
    k.copy_(src[1])
    w = torch.ones(d, device=DEV).bfloat16()
    want = QN.qk_norm_fwd(src[0], src[1], w, w, eps=1e-6)
    QN.qk_norm_fwd(q, k, w, w, eps=1e-6, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_same_bits_on_every_run_and_in_a_graph():
    q, k, dq, dk, wq, wk, cos, sin, _, _ = make(5000, 6, 2, 64, 64, 900, torch.bfloat16)
    call = lambda: (*QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6),  # noqa: E731
                    *QN.qk_norm_bwd(dq, dk, q, k, wq, wk, cos, sin, eps=1e-6))
    want = call()
    for a, b in zip(want, call()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        call()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = call()
            graphs.append((g, out))
    torch.cuda.current_stream().wait_stream(side)
    q.mul_(-1)
    want = [t.clone() for t in call()]
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        for a, b in zip(want, out):
            assert torch.equal(a, b)


def test_on_a_stream_of_its_own():
    q, k, _, _, wq, wk, cos, sin, _, _ = make(3000, 6, 6, 64, 64, 900, torch.bfloat16)
    want = QN.qk_norm_fwd(q, k, wq, wk, cos, sin, eps=1e-6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device=DEV)
        for _ in range(5):
            big = big @ big * 1e-3
        late = q + 0 * big.sum().clamp(-1, 1).nan_to_num().to(q.dtype)
        got = QN.qk_norm_fwd(late, k, wq, wk, cos, sin, eps=1e-6)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
