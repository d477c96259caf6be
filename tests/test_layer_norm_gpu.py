"""Layer norm against its formulas in 64 bits.

Tolerances: a result in type t is rounded once, by half a step of its value. Before that everything is fp32 (roundings of
U = 2^-24): sums over n columns are trees of depth log2 n behind at most n / 256 (wide rows: n / 1024) additions in a row, 24 + log2 n + n / 256
roundings with what goes into and comes out of them, of the sizes of the terms instead of the result. Sums over rows: as many
roundings as there are rows, of their absolute sum.
"""
import math

import pytest
import torch

from aeris_gb_b200.ops import layer_norm as LN

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
EPS = 1e-5


def half_step(dt):
    return torch.finfo(dt).eps / 2


def near(got, want, size, dt, roundings):
    slack = roundings * U * size
    bound = half_step(dt) * (want.abs() + slack) + slack + 1e-30
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (off / bound).max().item()


def rows_of(rows, cols, dt, layout, g):
    t = torch.randn((rows, cols), generator=g, device=DEV)
    if layout == "whole":
        return t.to(dt)
    gap = {"wider": 8, "odd pitch": 3, "odd start": 5}[layout]
    wide = torch.zeros((rows, cols + gap), device=DEV, dtype=dt)
    at = 1 if layout == "odd start" else 0
    wide[:, at:at + cols] = t.to(dt)
    return wide[:, at:at + cols]


def forward_check(x, w, b, y, stats):
    xd = x.double()
    n = x.shape[1]
    k = 24 + math.log2(n) + n / 256
    mean = xd.mean(1, keepdim=True)
    var = (xd - mean).square().mean(1, keepdim=True)
    rstd = (var + EPS).rsqrt()
    wd = 1.0 if w is None else w.double()
    bd = torch.zeros((), dtype=torch.float64, device=DEV) if b is None else b.double()
    level = xd.abs().mean(1, keepdim=True)
    size = (xd.abs() + level) * rstd * (1.0 if w is None else wd.abs()) + bd.abs()
    near(y, (xd - mean) * rstd * wd + bd, size, x.dtype, 2 * k)
    near(stats[:, :1], mean, level, torch.float32, k)
    # an error e of the mean adds e^2 to the variance
    near(stats[:, 1:], rstd, rstd * (1 + (k * U * level * rstd) ** 2), torch.float32, k)


def backward_check(dy, x, stats, w, dx, dw, db, base=0.0):
    xd, g = x.double(), dy.double()
    n, rows = x.shape[1], x.shape[0]
    k = 24 + math.log2(n) + n / 256
    mean, rstd = stats[:, :1].double(), stats[:, 1:].double()
    xhat, level = (xd - mean) * rstd, (xd.abs() + mean.abs()) * rstd
    gw = g if w is None else g * w.double()
    want = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
    size = rstd * (gw.abs() + gw.abs().mean(1, keepdim=True) + level * (gw.abs() * level).mean(1, keepdim=True))
    near(dx, want, size, x.dtype, 2 * k)
    if dw is not None:
        near(dw, base + (g * xhat).sum(0), abs(base) + (g.abs() * level).sum(0), torch.float32, rows + 16)
    if db is not None:
        near(db, base + g.sum(0), abs(base) + g.abs().sum(0), torch.float32, rows + 16)


SIZES = [(1, 1), (3, 2), (5, 7), (1, 16), (300, 17), (257, 64), (4, 96), (33, 127), (70, 128), (9, 129), (129, 256), (40, 333), (65, 512),
         (31, 513), (64, 768), (1, 1536), (77, 1536), (13, 2048), (11, 2049), (7, 4096), (6, 5120), (5, 8191), (4, 8200), (3, 16384),
         (2, 20001), (2000, 24)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["whole", "wider", "odd pitch", "odd start"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_both_directions(rows, cols, layout, dt):
    g = torch.Generator(device=DEV).manual_seed(rows * 31 + cols)
    x = rows_of(rows, cols, dt, layout, g)
    x += 2.0        # rows whose mean is not small
    dy = rows_of(rows, cols, dt, layout, g)
    w, b = (torch.randn(cols, generator=g, device=DEV).to(dt) for _ in range(2))
    y, stats = LN.layer_norm_fwd(x, w, b, eps=EPS)
    assert y.dtype is dt and stats.dtype is torch.float32
    forward_check(x, w, b, y, stats)
    dx, dw, db = LN.layer_norm_bwd(dy, x, stats, w)
    backward_check(dy, x, stats, w, dx, dw, db)


MANY = [(2400, 130), (2369, 257), (4000, 300), (2500, 513), (3001, 768), (2400, 1001), (2370, 1024), (2600, 1100), (2500, 1536), (2400, 1537),
        (2400, 2047), (2368, 2048), (9000, 640)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["whole", "wider", "odd pitch", "odd start"])
@pytest.mark.parametrize("rows,cols", MANY)
def test_many_rows(rows, cols, layout, dt):
    test_both_directions(rows, cols, layout, dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["whole", "odd pitch", "odd start"])
@pytest.mark.parametrize("rows,cols", [(1200, 3411), (1300, 5003), (1190, 8191), (400, 9001), (200, 16383), (330, 12544), (123, 290), (31, 4001),
                                       (33, 3968), (16, 8192), (2000, 65), (4096, 32)])
def test_wide_rows_and_clusters(rows, cols, layout, dt):
    test_both_directions(rows, cols, layout, dt)


@pytest.mark.parametrize("rows,cols", [(65, 512), (40, 333), (77, 1536), (5, 8191), (900, 48), (2500, 640), (2400, 333)])
@pytest.mark.parametrize("parts", ["none", "weight", "bias", "fp32"])
def test_weight_and_bias_may_be_missing_or_in_fp32(rows, cols, parts):
    g = torch.Generator(device=DEV).manual_seed(3)
    x, dy = (rows_of(rows, cols, torch.bfloat16, "whole", g) for _ in range(2))
    w, b = (torch.randn(cols, generator=g, device=DEV) for _ in range(2))
    if parts != "fp32":
        w, b = (w.bfloat16() if parts == "weight" else None), (b.bfloat16() if parts == "bias" else None)
    y, stats = LN.layer_norm_fwd(x, w, b, eps=EPS)
    forward_check(x, w, b, y, stats)
    dx, dw, db = LN.layer_norm_bwd(dy, x, stats, w, bias=b is not None)
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    backward_check(dy, x, stats, w, dx, dw, db)


@pytest.mark.parametrize("rows,cols", [(65, 512), (40, 333), (77, 1536), (5, 9000), (900, 48), (2500, 640), (2400, 333), (1300, 4999),
                                       (1250, 3411), (300, 16001), (20, 4000), (12, 6144)])
def test_places_that_are_given(rows, cols):
    g = torch.Generator(device=DEV).manual_seed(4)
    x, dy = (rows_of(rows, cols, torch.bfloat16, "whole", g) for _ in range(2))
    w, b = (torch.randn(cols, generator=g, device=DEV).bfloat16() for _ in range(2))
    y, stats = LN.layer_norm_fwd(x, w, b, eps=EPS)
    # in place, and with rows and columns around the results that stay as they were
    x2 = x.clone()
    place = torch.full((rows + 2, 2), 7.0, device=DEV)
    y2, stats2 = LN.layer_norm_fwd(x2, w, b, eps=EPS, out=x2, stats=place[1:rows + 1])
    assert y2 is x2 and torch.equal(y2, y) and torch.equal(stats2, stats)
    assert bool((place[0] == 7).all()) and bool((place[-1] == 7).all())
    wide = torch.full((rows + 2, cols + 9), 3.0, device=DEV, dtype=torch.bfloat16)
    y3, _ = LN.layer_norm_fwd(x, w, b, eps=EPS, out=wide[1:-1, 5:-4])
    forward_check(x, w, b, y3, stats)         # rows that start elsewhere may be added up in another order
    wide[1:-1, 5:-4] = 3.0
    assert bool((wide == 3).all())
    dx, dw, db = LN.layer_norm_bwd(dy, x, stats, w)
    for over in ("dy", "x"):
        args = {"dy": dy.clone(), "x": x.clone()}
        dw2, db2 = (torch.full((cols,), 0.5, device=DEV) for _ in range(2))
        dx2, *_ = LN.layer_norm_bwd(args["dy"], args["x"], stats, w, dx=args[over], dw=dw2, db=db2)
        assert dx2 is args[over] and torch.equal(dx2, dx)
        backward_check(dy, x, stats, w, dx2, dw2, db2, base=0.5)


def test_no_rows():
    x = torch.empty((0, 64), device=DEV, dtype=torch.bfloat16)
    w = torch.ones(64, device=DEV)
    y, stats = LN.layer_norm_fwd(x, w, w, eps=EPS)
    assert y.shape == (0, 64) and stats.shape == (0, 2)
    dx, dw, db = LN.layer_norm_bwd(x, x, stats, w)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_rows_that_are_not_finite_stay_by_themselves():
    x = torch.randn((9, 640), device=DEV)
    clean, _ = LN.layer_norm_fwd(x, eps=EPS)
    x[2, 5], x[4, 600] = math.inf, math.nan
    y, _ = LN.layer_norm_fwd(x, eps=EPS)
    others = [0, 1, 3, 5, 6, 7, 8]
    assert torch.equal(y[others], clean[others]) and y[2].isnan().any() and y[4].isnan().all()


def test_large_mean():
    """Rows around 1000 with a spread of one: a difference of two large sums would leave three digits."""
    g = torch.Generator(device=DEV).manual_seed(5)
    for cols in (100, 1536, 9000):
        x = 1000 + torch.randn((17, cols), generator=g, device=DEV)
        y, stats = LN.layer_norm_fwd(x, eps=EPS)
        forward_check(x, None, None, y, stats)


def test_captured_and_on_another_stream():
    g = torch.Generator(device=DEV).manual_seed(6)
    x, dy = (rows_of(500, 768, torch.bfloat16, "whole", g) for _ in range(2))
    w = torch.randn(768, generator=g, device=DEV)

    def both():
        y, stats = LN.layer_norm_fwd(x, w, w, eps=EPS)
        return (y, stats, *LN.layer_norm_bwd(dy, x, stats, w))

    want = [t.clone() for t in both()]
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


def test_gradient_against_differences():
    g = torch.Generator(device=DEV).manual_seed(7)
    x, dy, v = (torch.randn((6, 200), generator=g, device=DEV) for _ in range(3))
    w, b = (torch.randn(200, generator=g, device=DEV) for _ in range(2))
    y, stats = LN.layer_norm_fwd(x, w, b, eps=EPS)
    dx, dw, db = LN.layer_norm_bwd(dy, x, stats, w)
    # central differences over h = 2^-5: the third derivative's part is of the size h^2 |v|^3, a few 1e-3 of the slope's terms
    h = 2.0 ** -5
    up, down = (LN.layer_norm_fwd(x + s * h * v, w, b, eps=EPS)[0].double() for s in (1, -1))
    slope = ((up - down) / (2 * h) * dy.double()).sum(1)
    terms = (dy.double().abs() * (w.abs() * v.abs() * stats[:, 1:]).double()).sum(1)
    assert bool(((dx.double() * v.double()).sum(1) - slope).abs().lt(4e-3 * terms).all())
    up, down = (LN.layer_norm_fwd(x, w + s * h * v[0], b + s * h * v[1], eps=EPS)[0].double() for s in (1, -1))
    slope = ((up - down) / (2 * h) * dy.double()).sum()
    assert abs(float((dw.double() * v[0].double()).sum() + (db.double() * v[1].double()).sum() - slope)) < 1e-4 * float(terms.sum())


@pytest.mark.parametrize("cols", [64, 333, 1536, 9000])
def test_same_bits_on_every_run(cols):
    x, dy = (torch.randn((2777, cols), device=DEV).bfloat16() for _ in range(2))
    w = torch.randn(cols, device=DEV)
    first = LN.layer_norm_bwd(dy, x, LN.layer_norm_fwd(x, w, eps=EPS)[1], w)
    for _ in range(5):
        again = LN.layer_norm_bwd(dy, x, LN.layer_norm_fwd(x, w, eps=EPS)[1], w)
        assert all(map(torch.equal, again, first))


def test_offsets_past_32_bits():
    """Rows further than 2^31 elements apart from the first, out of one large matrix (4.3 GB)."""
    wide = torch.empty((2 ** 16 + 1, 2 ** 15 + 64), device=DEV, dtype=torch.bfloat16)
    x = wide[:, 64:64 + 96]
    x.copy_(torch.randn(x.shape, device=DEV))
    y, stats = LN.layer_norm_fwd(x, eps=EPS, out=x)
    z, again = LN.layer_norm_fwd(y.contiguous(), eps=EPS)
    assert float((y[-1].float() - z[-1].float()).abs().max()) < 0.05
    dx, _, db = LN.layer_norm_bwd(y, y, again)
    backward_check(y[-50:], y[-50:], again[-50:], None, dx[-50:], None, None)
    assert bool((db.double() - y.double().sum(0)).abs().lt((2 ** 16 + 17) * U * y.double().abs().sum(0)).all())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 5), (7, 64), (300, 333), (2500, 333), (1300, 1001), (40, 1536), (1200, 3411), (330, 12544), (30, 20001)])
@pytest.mark.parametrize("gap,start", [(8, 0), (3, 0), (8, 1)])
def test_what_lies_between_rows_is_not_read_into_results(rows, cols, gap, start, dt):
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    x, dy = (torch.full((rows, cols + gap), math.nan, device=DEV, dtype=dt)[:, start:start + cols] for _ in range(2))
    for t in (x, dy):
        t.copy_(torch.randn((rows, cols), generator=g, device=DEV))
    w, b = (torch.randn(cols, generator=g, device=DEV) for _ in range(2))
    y, stats = LN.layer_norm_fwd(x, w, b, eps=EPS)
    forward_check(x, w, b, y, stats)
    backward_check(dy, x, stats, w, *LN.layer_norm_bwd(dy, x, stats, w))
