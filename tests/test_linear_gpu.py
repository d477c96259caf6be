"""Linear layers with bias, activation and residual against their formulas in 64 bits.

Tolerances: products of bf16 are exact in fp32; the tensor core adds 16 of them at a time and truncates, so that a sum over K has at
most K / 16 + 8 errors of a step, 2^-23, of its terms' absolute sum. Activations have slopes up to 1.13, are a few operations
with approximate exponentials and reciprocals (2^-19 of 1 + |z| is allowed for), and results are rounded once, by half a step. The
gradient of z goes into the products in bf16: half a step of every term.
"""
import math

import pytest
import torch

from aeris_gb_b200.ops import linear as LI

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8          # half a step of bf16
BF = torch.bfloat16


def step_sum(k):
    return (k / 16 + 8) * 2.0 ** -23


def act64(z, act):
    """(value, slope)"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if act == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * (-z * z / 2).exp() / math.sqrt(2 * math.pi)
    p = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z * p, p + z * p * (1 - p) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)


def within(got, want, bound):
    off = (got.double() - want).abs()
    assert bool((off <= bound + 1e-30).all()), (off / (bound + 1e-30)).max().item()


def forward_check(x, w, b, act, resid, y, z):
    xd, wd = x.double(), w.double()
    zd, size = xd @ wd.T, xd.abs() @ wd.abs().T
    if b is not None:
        zd, size = zd + b.double(), size + b.double().abs()
    ez = step_sum(x.shape[1]) * size
    if z is not None:
        within(z, zd, HALF * (zd.abs() + ez) + ez)
    f, _ = act64(zd, act)
    ef = 1.13 * ez + (0 if act in ("none", "relu") else 2.0 ** -19 * (1 + zd.abs()))
    r = 0 if resid is None else resid.double()
    yd = f + r
    ef = ef + 2.0 ** -23 * (f.abs() + (0 if resid is None else r.abs()))
    within(y, yd, HALF * (yd.abs() + ef) + ef)


def backward_check(dy, x, w, z, act, dx, dw, db, base=0.0):
    slope = act64(z.double(), act)[1] if z is not None else 1.0
    d = dy.double()
    dz = d * slope
    # z = +-0 aside, a slope is off by the approximations only
    e_dz = 0 if act in ("none", "relu") else d.abs() * 2.0 ** -19 * (2 + z.double().abs())
    e_in = e_dz + (0 if act == "none" else HALF * (dz.abs() + e_dz))
    rows, cols = dy.shape
    if dx is not None:
        want = dz @ w.double()
        e = e_in @ w.double().abs() if act != "none" else 0
        e = e + step_sum(cols) * ((dz.abs() * 1.01) @ w.double().abs())
        within(dx, want, HALF * (want.abs() + e) + e)
    if dw is not None:
        want = base + dz.T @ x.double()
        e = e_in.T @ x.double().abs() if act != "none" else 0
        e = e + step_sum(rows) * ((dz.abs() * 1.01).T @ x.double().abs() + abs(base))
        within(dw, want, (HALF * (want.abs() + e) if dw.dtype is BF else 2.0 ** -24 * want.abs()) + e)
    if db is not None:
        e = (e_dz + (rows + 16) * 2.0 ** -24 * dz.abs()).sum(0) + 2.0 ** -23 * abs(base)
        within(db, base + dz.sum(0), e)


def rnd(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def laid_out(t, layout):
    if layout == "whole":
        return t.to(BF)
    rows, cols = t.shape
    gap, at = {"wider": (16, 8), "odd pitch": (3, 0), "odd start": (8, 1)}[layout]
    wide = torch.zeros((rows, cols + gap), device=DEV, dtype=BF)
    wide[:, at:at + cols] = t.to(BF)
    return wide[:, at:at + cols]


SIZES = [(1, 1, 1), (1, 64, 64), (1, 1536, 4096), (2, 3, 5), (3, 1000, 70), (4, 300, 1), (5, 2000, 33), (6, 48, 500), (7, 8, 16), (8, 512, 333),
         (8, 5120, 40), (9, 256, 256), (17, 100, 31), (33, 333, 777), (64, 64, 32), (100, 40, 130), (127, 65, 129),
         (128, 128, 128), (129, 256, 33), (200, 520, 256), (256, 512, 512), (300, 1000, 264), (513, 96, 1000), (1000, 777, 320),
         (2500, 128, 640), (5000, 48, 200)]


@pytest.mark.parametrize("rows,inner,cols", SIZES)
@pytest.mark.parametrize("act", LI.ACTIVATIONS)
def test_both_directions(rows, inner, cols, act):
    g = torch.Generator(device=DEV).manual_seed(rows + 7 * inner + 13 * cols)
    x, w = rnd(g, rows, inner).to(BF), (rnd(g, cols, inner) / math.sqrt(inner)).to(BF)
    b, resid = rnd(g, cols), rnd(g, rows, cols).to(BF)
    y, z = LI.linear_fwd(x, w, b, act=act, resid=resid, keep=True)
    forward_check(x, w, b, act, resid, y, z)
    dy = rnd(g, rows, cols).to(BF)
    backward_check(dy, x, w, z if act != "none" else None, act, *LI.linear_bwd(dy, x, w, z, act=act))


@pytest.mark.parametrize("layout", ["whole", "wider", "odd pitch", "odd start"])
@pytest.mark.parametrize("rows,inner,cols", [(1, 40, 24), (65, 200, 136), (300, 72, 264), (130, 77, 99)])
def test_layouts_of_inputs_and_results(rows, inner, cols, layout):
    g = torch.Generator(device=DEV).manual_seed(rows)
    x, w, resid, dy = (laid_out(rnd(g, *s), layout) for s in ((rows, inner), (cols, inner), (rows, cols), (rows, cols)))
    b = rnd(g, cols + 1)[1:].to(BF)
    out, kept = (laid_out(torch.zeros(rows + 2, cols, device=DEV), layout) for _ in range(2))
    for t in (out, kept):
        t.fill_(5.0)
    y, z = LI.linear_fwd(x, w, b, act="silu", resid=resid, keep=True, out=out[1:-1], z=kept[1:-1])
    assert y.data_ptr() == out[1:-1].data_ptr() and z.data_ptr() == kept[1:-1].data_ptr()
    for t in (out, kept):
        assert bool((t[0] == 5).all()) and bool((t[-1] == 5).all())
    forward_check(x, w, b, "silu", resid, y, z)
    place = laid_out(torch.zeros(rows, inner, device=DEV), layout)
    dw, db = torch.full((cols, inner + 3), 2.0, device=DEV)[:, :inner], torch.full((cols,), 2.0, device=DEV)
    dx, dw2, db2 = LI.linear_bwd(dy, x, w, z, act="silu", dx=place, dw=dw, db=db)
    assert dx is place and dw2 is dw and db2 is db
    backward_check(dy, x, w, z, "silu", dx, dw, db, base=2.0)


def test_a_single_row_without_a_pitch():
    g = torch.Generator(device=DEV).manual_seed(11)
    x, w, r = rnd(g, 72).to(BF).expand(1, 72), rnd(g, 72).to(BF).expand(1, 72), rnd(g, 1).to(BF).expand(1, 1)
    y, z = LI.linear_fwd(x, w, resid=r, keep=True, act="silu", out=torch.empty(1, device=DEV, dtype=BF).expand(1, 1))
    forward_check(x, w, None, "silu", r, y, z)
    backward_check(r, x, w, z, "silu", *LI.linear_bwd(r, x, w, z, act="silu", dx=torch.empty(72, device=DEV, dtype=BF).expand(1, 72)))
    many = rnd(g, 40, 72).to(BF)
    y, z = LI.linear_fwd(many, w, keep=True)
    forward_check(many, w, None, "none", None, y, z)


def test_columns_beside_a_result_stay():
    g = torch.Generator(device=DEV).manual_seed(1)
    x, w = rnd(g, 100, 64).to(BF), rnd(g, 88, 64).to(BF)
    wide = torch.full((100, 128), 9.0, device=DEV, dtype=BF)
    for at in (8, 3):
        y, _ = LI.linear_fwd(x, w, out=wide[:, at:at + 88])
        forward_check(x, w, None, "none", None, y, None)
        wide[:, at:at + 88] = 9.0
        assert bool((wide == 9).all())


def test_result_in_the_place_of_the_residual():
    g = torch.Generator(device=DEV).manual_seed(2)
    x, w, r = rnd(g, 700, 320).to(BF), rnd(g, 1000, 320).to(BF), rnd(g, 700, 1000).to(BF)
    want, none = LI.linear_fwd(x, w, act="relu", resid=r)
    assert none is None
    got, _ = LI.linear_fwd(x, w, act="relu", resid=r, out=r)
    assert got is r and torch.equal(got, want)


def test_gradients_by_choice():
    g = torch.Generator(device=DEV).manual_seed(3)
    x, w, z, dy = rnd(g, 90, 64).to(BF), rnd(g, 50, 64).to(BF), rnd(g, 90, 50).to(BF), rnd(g, 90, 50).to(BF)
    full = LI.linear_bwd(dy, x, w, z, act="gelu")
    for need_dx in (False, True):
        for need_dw in (False, True):
            for bias in (False, True):
                got = LI.linear_bwd(dy, x, w, z, act="gelu", need_dx=need_dx, need_dw=need_dw, bias=bias)
                for t, u, wanted in zip(got, full, (need_dx, need_dw, bias)):
                    assert (t is None) == (not wanted) and (t is None or torch.equal(t, u))


def test_no_rows():
    x, w = torch.empty((0, 16), device=DEV, dtype=BF), torch.ones((8, 16), device=DEV, dtype=BF)
    y, z = LI.linear_fwd(x, w, keep=True)
    assert y.shape == (0, 8) and z.shape == (0, 8)
    dx, dw, db = LI.linear_bwd(y, x, w)
    assert dx.shape == (0, 16) and not dw.any() and not db.any()
    dw, db = torch.full((8, 16), 3.0, device=DEV), torch.full((8,), 3.0, device=DEV)
    LI.linear_bwd(y, x, w, dw=dw, db=db)
    assert bool((dw == 3).all()) and bool((db == 3).all())


@pytest.mark.parametrize("act", LI.ACTIVATIONS)
def test_far_values(act):
    """Activations and their slopes where exponentials leave the range of fp32, through an identity."""
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 12.0, -12.0, 90.0, -90.0, 700.0, -700.0, 1e18, -1e18, 1e30, -1e30, 3e38, -3e38], device=DEV)
    x, w = torch.diag(v).to(BF), torch.eye(16, device=DEV, dtype=BF)
    z64 = x.double()
    y, z = LI.linear_fwd(x, w, act=act, keep=True)
    assert torch.equal(z, x) or torch.equal(z.float(), x.float() + 0.0)
    # the square or cube of a far value is infinite in 64 bits' formula as well: 0 and 1 are meant
    lim = z64.clamp(-1e3, 1e3)
    f, s = act64(lim, act)
    f = torch.where(z64.abs() > 1e3, z64 * (f / torch.where(lim == 0, 1.0, lim)), f)
    within(y, f, HALF * f.abs() + 2.0 ** -19)
    dy = torch.ones((16, 16), device=DEV, dtype=BF)
    # dw = dz^T x needs finite rows: dx through the identity shows dz itself
    dx, _, _ = LI.linear_bwd(dy, x, w, x, act=act, need_dw=False, bias=False)
    within(dx, s, 2 * HALF * s.abs() + 2.0 ** -18)


def test_values_that_are_not_finite_stay_in_their_row():
    g = torch.Generator(device=DEV).manual_seed(4)
    x, w = rnd(g, 150, 96).to(BF), rnd(g, 70, 96).to(BF)
    clean, _ = LI.linear_fwd(x, w, act="gelu")
    x[149, 3], x[5, 95] = math.nan, math.inf
    y, _ = LI.linear_fwd(x, w, act="gelu")
    rest = [i for i in range(150) if i not in (5, 149)]
    assert torch.equal(y[rest], clean[rest]) and y[149].isnan().all() and not y[5].isfinite().all()


def test_broadcast_rows():
    g = torch.Generator(device=DEV).manual_seed(5)
    x, w = rnd(g, 1, 64).to(BF).expand(200, 64), rnd(g, 48, 64).to(BF)
    r, dy = rnd(g, 1, 48).to(BF).expand(200, 48), rnd(g, 1, 48).to(BF).expand(200, 48)
    y, z = LI.linear_fwd(x, w, act="silu", resid=r, keep=True)
    forward_check(x, w, None, "silu", r, y, z)
    backward_check(dy, x, w, z, "silu", *LI.linear_bwd(dy, x, w, z, act="silu"))
    backward_check(dy, x, w, None, "none", *LI.linear_bwd(dy, x, w))


@pytest.mark.parametrize("rows,inner,cols", [(300, 264, 520), (4000, 256, 512), (77, 33, 65)])
def test_same_bits_captured_and_on_another_stream(rows, inner, cols):
    g = torch.Generator(device=DEV).manual_seed(6)
    x, w, dy = rnd(g, rows, inner).to(BF), rnd(g, cols, inner).to(BF), rnd(g, rows, cols).to(BF)
    b = rnd(g, cols)

    def both():
        y, z = LI.linear_fwd(x, w, b, act="gelu", keep=True)
        return (y, z, *LI.linear_bwd(dy, x, w, z, act="gelu"))

    want = [t.clone() for t in both()]
    for _ in range(3):
        assert all(map(torch.equal, both(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(map(torch.equal, got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(map(torch.equal, got, want))


def test_two_calls_at_once():
    g = torch.Generator(device=DEV).manual_seed(7)
    sets = [(rnd(g, 1000, 512).to(BF), rnd(g, 768, 512).to(BF), rnd(g, 1000, 768).to(BF)) for _ in range(2)]
    want = [LI.linear_bwd(dy, x, w, dy, act="silu") for x, w, dy in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(5):
        for i, (s, (x, w, dy)) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[i] = LI.linear_bwd(dy, x, w, dy, act="silu")
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p, q in zip(got, want) for a, b in zip(p, q))


def test_gradient_against_differences():
    """One column of x moved by a step that bf16 holds: the fp32 sum of the results' differences against dx."""
    g = torch.Generator(device=DEV).manual_seed(8)
    x = (rnd(g, 16, 64) * 8).round().to(BF) / 8
    w = (rnd(g, 32, 64) / 8).to(BF)
    for act in LI.ACTIVATIONS:
        if act == "relu":
            continue          # not smooth
        h = 2.0 ** -4
        up, down = (LI.linear_fwd((x.float() + s * h * (torch.arange(64, device=DEV) == 5)).to(BF), w, act=act, keep=True)[0].double()
                    for s in (1, -1))
        _, z = LI.linear_fwd(x, w, act=act, keep=True)
        dy = torch.ones((16, 32), device=DEV, dtype=BF)
        dx, _, _ = LI.linear_bwd(dy, x, w, z, act=act)
        slope = ((up - down) / (2 * h)).sum(1)
        # results are rounded to bf16 (half a step of each, over the step), third derivatives below 1, z and dz in bf16
        bound = (HALF * (up.abs() + down.abs()) / (2 * h)).sum(1) + (w[:, 5].double().abs() ** 3).sum() * h * h + \
            2 * HALF * (w[:, 5].double().abs() * (1 + z.double().abs())).sum(1) + HALF * slope.abs()
        assert bool((dx[:, 5].double() - slope).abs().le(bound).all()), act


def test_offsets_past_32_bits():
    """Rows further than 2^31 elements behind the first of x and of the result (4.3 GB each)."""
    rows, inner, cols = 2 ** 16 + 130, 2 ** 15 + 8, 2 ** 15 + 24
    x = torch.empty((rows, inner), device=DEV, dtype=BF)[:, :64]
    g = torch.Generator(device=DEV).manual_seed(9)
    x.copy_(rnd(g, rows, 64))
    w = rnd(g, 40, 64).to(BF)
    y = torch.empty((rows, cols), device=DEV, dtype=BF)[:, :40]
    LI.linear_fwd(x, w, act="gelu", out=y)
    forward_check(x[-200:], w, None, "gelu", None, y[-200:], None)
    dx, dw, db = LI.linear_bwd(y, x, w)
    backward_check(y[-200:], x[-200:], w, None, "none", dx[-200:], None, None)
    backward_check(y, x, w, None, "none", None, dw, db)


def place(rows, cols, pitch, value=7.0):
    """A matrix whose rows start on 16-byte boundaries, and what lies between and behind them."""
    buf = torch.full((rows * pitch + 64,), value, device=DEV, dtype=BF)
    inside = torch.zeros_like(buf, dtype=torch.bool)
    inside[:rows * pitch].view(rows, pitch)[:, :cols] = True
    return buf[:rows * pitch].view(rows, pitch)[:, :cols], buf, ~inside


@pytest.mark.parametrize("cols", [1, 35, 70, 100, 147, 1015, 2047])
@pytest.mark.parametrize("rows,inner", [(1, 25000), (10, 48), (64, 512), (200, 512), (1035, 96), (3000, 512), (9000, 264)])
def test_rows_that_end_between_16_byte_boundaries_leave_what_lies_behind(rows, inner, cols):
    """Results whose rows start on 16-byte boundaries, of any width: the elements up to the next boundary are not theirs."""
    g = torch.Generator(device=DEV).manual_seed(rows + inner + cols)
    x, w, b = rnd(g, rows, inner).to(BF), (rnd(g, cols, inner) / math.sqrt(inner)).to(BF), rnd(g, cols)
    r = rnd(g, rows, cols).to(BF)
    for pitch in ((cols + 7) // 8 * 8, (cols + 7) // 8 * 8 + 8):
        (out, ob, out_rest), (z, zb, z_rest) = (place(rows, cols, pitch) for _ in range(2))
        out.copy_(r)                                   # the residual is the result's place
        LI.linear_fwd(x, w, b, act="gelu", resid=out, keep=True, out=out, z=z)
        forward_check(x, w, b, "gelu", r, out, z)
        assert bool((ob[out_rest] == 7).all()) and bool((zb[z_rest] == 7).all())
        y, _ = LI.linear_fwd(x, w, b, act="gelu", resid=r, out=place(rows, cols, pitch)[0])
        assert torch.equal(y, out)
        # of dx: dy [rows, inner], w [inner, cols]
        dy, xx, ww = rnd(g, rows, inner).to(BF), rnd(g, rows, cols).to(BF), (rnd(g, inner, cols) / math.sqrt(inner)).to(BF)
        for need_dw in (False, True):
            dx, gb, dx_rest = place(rows, cols, pitch)
            _, dw, db = LI.linear_bwd(dy, xx, ww, dx=dx, need_dw=need_dw)
            backward_check(dy, xx, ww, None, "none", dx, dw, db)
            assert bool((gb[dx_rest] == 7).all())


@pytest.mark.parametrize("rows,inner,cols", [(1, 35, 70), (5, 100, 33), (10, 48, 147), (200, 295, 100), (1035, 515, 777), (3000, 70, 1015), (9000, 333, 260)])
@pytest.mark.parametrize("gap", [0, 8, 3])
def test_what_lies_between_rows_is_not_read_into_results(rows, inner, cols, gap):
    g = torch.Generator(device=DEV).manual_seed(rows + inner + cols + gap)

    def of(r, c):
        t, buf, rest = place(r, c, (c + 7) // 8 * 8 + gap, math.nan)
        t.copy_(rnd(g, r, c))
        return t

    x, w, dy, resid, z = of(rows, inner), of(cols, inner), of(rows, cols), of(rows, cols), of(rows, cols)
    w.mul_(1 / math.sqrt(inner))
    b = rnd(g, cols)
    y, kept = LI.linear_fwd(x, w, b, act="silu", resid=resid, keep=True)
    forward_check(x, w, b, "silu", resid, y, kept)
    for act, zz in (("silu", z), ("none", None)):
        dx, dw, db = LI.linear_bwd(dy, x, w, zz, act=act)
        backward_check(dy, x, w, zz, act, dx, dw, db)
