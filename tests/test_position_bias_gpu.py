"""Window attention with a position bias against its formulas in 64 bits.

Tolerances. Scores: products of bf16 are exact in fp32; the tensor core truncates after every 16 of them (d / 16 + 4 errors of 2^-23 of the terms'
absolute sum), the bias and the statistics add roundings of 2^-23 of their sizes: es, the error of a score, which is the
relative error of its probability (2^-21 more for the exponential). Probabilities and ds go into products in bf16: half a step, 2^-8, of
each term. Results in bf16 are rounded once more. delta comes from the rounded o in the dQ kernel (dO times the error of o);
the others have it exactly but for fp32. The table's gradient is fp32 throughout: of every ds the error of p and of dp - delta.
"""
import math

import pytest
import torch

from aeris_gb_b200.ops import attention as A
from aeris_gb_b200.ops import position_bias as PB

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
HALF = 2.0 ** -8
LOG2E = 1 / math.log(2)


def index_of(window, buckets):
    h, w = window
    t = torch.arange(h * w, device=DEV)
    y, x = t // w, t % w
    at = (y[:, None] - y + h - 1) * (2 * w - 1) + x[:, None] - x + w - 1
    return at if buckets is None else buckets.long()[at]


def heads_of(t, n, heads, d, parts=1):
    return t.double().reshape(-1, n, parts, heads, d).permute(2, 0, 3, 1, 4)


def formula(qkv, window, heads, d, table, buckets, scale):
    n = window[0] * window[1]
    q, k, v = heads_of(qkv, n, heads, d, 3)
    index = index_of(window, buckets)
    bias = table.double()[index].permute(2, 0, 1)
    bias = torch.where(bias <= PB.HIDDEN, -math.inf, bias)
    s = scale * (q @ k.transpose(-1, -2)) + bias
    lse = torch.logsumexp(s, -1, keepdim=True)
    lse = torch.where(lse == -math.inf, math.inf, lse)
    p = (s - lse).exp()
    fin = torch.where(bias.isfinite(), bias.abs(), 0.0)
    es = (d / 16 + 4) * 2.0 ** -23 * abs(scale) * (q.abs() @ k.abs().transpose(-1, -2)) + \
        2.0 ** -22 * (fin + torch.where(lse.isfinite(), lse.abs(), 0.0) + 8)
    return q, k, v, p, lse.squeeze(-1), es + 2.0 ** -21, index


def within(got, want, bound):
    off = (got.double() - want).abs()
    assert bool((off <= bound + 1e-30).all()), (off / (bound + 1e-30)).max().item()


def together(x):
    return x.permute(0, 2, 1, 3).flatten(2).flatten(0, 1)


def forward_check(o, lse, f):
    q, k, v, p, want, es, _ = f
    size = p @ v.abs()
    e = HALF * size + (2 * es * p) @ v.abs() + (p.shape[-1] / 16 + 8) * 2.0 ** -23 * size
    within(o, together(p @ v), together(HALF * ((p @ v).abs() + e) + e))
    seen = want.isfinite()
    assert torch.equal(lse.isinf() & (lse > 0), ~seen)
    es = es.amax(-1)
    within(lse[seen], want[seen] * LOG2E, (es * LOG2E + 2.0 ** -21 * (1 + want.abs() * LOG2E))[seen])


def backward_check(d_o, o, dqkv, dtable, f, window, heads, d, scale, table_rows, base=0.0):
    q, k, v, p, _, es, index = f
    n = window[0] * window[1]
    do, og = heads_of(d_o, n, heads, d)[0], heads_of(o, n, heads, d)[0]
    dp = do @ v.transpose(-1, -2)
    dp_size = do.abs() @ v.abs().transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_dp = (d / 16 + 4) * 2.0 ** -23 * dp_size
    e_p = 2 * es * p
    # fp32 delta: sums of p dp, of e_p |dp - delta|
    e_delta = (p * e_dp + e_p * (dp - delta).abs()).sum(-1, keepdim=True) + (n / 16 + 16) * 2.0 ** -23 * (p * dp_size).sum(-1, keepdim=True)
    e_o = (do * (og - p @ v)).sum(-1, keepdim=True).abs() + d * 2.0 ** -23 * (do.abs() * og.abs()).sum(-1, keepdim=True)
    e_ds = e_p * (dp - delta).abs() + p * (e_dp + e_delta) + 2.0 ** -22 * ds.abs()
    trunc = (n / 16 + 8) * 2.0 ** -23
    c = abs(scale)
    want_q, want_k, want_v = scale * (ds @ k), scale * (ds.transpose(-1, -2) @ q), p.transpose(-1, -2) @ do
    e_in = HALF * (ds.abs() + e_ds) + e_ds
    eq = c * ((e_in + 1.01 * p * e_o + trunc * ds.abs()) @ k.abs())
    ek = c * ((e_in + trunc * ds.abs()).transpose(-1, -2) @ q.abs())
    ev = (HALF * p + e_p + trunc * p).transpose(-1, -2) @ do.abs()
    for i, (w, e) in enumerate(((want_q, eq), (want_k, ek), (want_v, ev))):
        got = dqkv[:, i * heads * d:(i + 1) * heads * d]
        within(got, together(w), together(HALF * (w.abs() + e) + e))
    if dtable is not None:
        at = index.reshape(-1)
        zero = torch.zeros((table_rows, heads), dtype=torch.float64, device=DEV)
        want = zero.index_add(0, at, ds.sum(0).flatten(1).T) + base
        # sums over windows one after the other, over pairs in parts: as many roundings as there are of both, of the terms
        terms = ds.shape[0] + n / 8 + 64
        e = zero.index_add(0, at, (e_ds + terms * 2.0 ** -24 * ds.abs()).sum(0).flatten(1).T) + 2.0 ** -23 * abs(base)
        within(dtable, want, e + 2.0 ** -23 * want.abs())


def coarse(window, rows, g):
    """Buckets at random, each relative position its own; bucket 0 is hidden by some tables below."""
    return torch.randint(0, rows, (PB.relative_positions(window),), generator=g, device=DEV, dtype=torch.int32)


def make(n_win, window, heads, d, g, table_rows=None, dt=torch.float32, strength=1.0):
    n = window[0] * window[1]
    qkv = torch.randn((n_win * n, 3 * heads * d), generator=g, device=DEV).to(BF)
    buckets = None if table_rows is None else coarse(window, table_rows, g)
    table = (strength * torch.randn((table_rows or PB.relative_positions(window), heads), generator=g, device=DEV)).to(dt)
    d_o = torch.randn((n_win * n, heads * d), generator=g, device=DEV).to(BF)
    return qkv, table, buckets, d_o


def run_both(qkv, table, buckets, d_o, n_win, window, heads, d, scale=None):
    o, lse = PB.biased_attn_fwd(qkv, n_win, window, heads, d, table, buckets, scale=scale)
    dqkv, dtable = PB.biased_attn_bwd(d_o, qkv, o, lse, n_win, window, heads, d, table, buckets, scale=scale)
    f = formula(qkv, window, heads, d, table, buckets, 1 / math.sqrt(d) if scale is None else scale)
    forward_check(o, lse, f)
    backward_check(d_o, o, dqkv, dtable, f, window, heads, d, 1 / math.sqrt(d) if scale is None else scale, table.shape[0])
    return o, lse, dqkv, dtable


WINDOWS = [(1, (1, 1)), (3, (1, 2)), (2, (1, 17)), (2, (31, 1)), (5, (4, 4)), (7, (8, 8)), (2, (9, 7)), (3, (8, 12)), (2, (5, 19)), (1, (1, 127)),
           (2, (8, 16)), (2, (3, 43)), (1, (12, 16)), (2, (13, 17)), (1, (15, 17)), (3, (16, 16)), (1, (2, 150)), (1, (1, 384)), (2, (30, 30))]


@pytest.mark.parametrize("heads,d", [(2, 32), (3, 64), (1, 128), (2, 72), (1, 8)])
@pytest.mark.parametrize("n_win,window", WINDOWS)
def test_both_directions(n_win, window, heads, d):
    g = torch.Generator(device=DEV).manual_seed(n_win + 3 * window[0] + 5 * window[1] + d)
    run_both(*make(n_win, window, heads, d, g), n_win, window, heads, d)


@pytest.mark.parametrize("dt,wide", [(torch.float32, torch.int32), (BF, torch.int64)])
@pytest.mark.parametrize("n_win,window,heads,d,rows", [(3, (8, 8), 5, 40, 1), (2, (9, 13), 33, 16, 7), (4, (10, 20), 2, 96, 40), (150, (4, 6), 2, 64, 5)])
def test_buckets(n_win, window, heads, d, rows, dt, wide):
    g = torch.Generator(device=DEV).manual_seed(rows)
    qkv, table, buckets, d_o = make(n_win, window, heads, d, g, rows, dt)
    run_both(qkv, table, buckets.to(wide), d_o, n_win, window, heads, d)


def test_zero_table_is_plain_attention():
    g = torch.Generator(device=DEV).manual_seed(0)
    qkv, table, _, d_o = make(3, (14, 10), 4, 64, g)
    o, lse = PB.biased_attn_fwd(qkv, 3, (14, 10), 4, 64, 0 * table)
    want, want_lse = A.attn_fwd(qkv, 3, 140, 4, 64)
    assert float((o.float() - want.float()).norm() / want.float().norm()) < 2 * HALF
    assert float((lse - want_lse).abs().max()) < 1e-4
    dqkv, _ = PB.biased_attn_bwd(d_o, qkv, o, lse, 3, (14, 10), 4, 64, 0 * table)
    want = A.attn_bwd(qkv, o, d_o, lse, 3, 140, 4, 64)
    assert float((dqkv.float() - want.float()).norm() / want.float().norm()) < 2 * HALF


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min, -1e30])
@pytest.mark.parametrize("window", [(6, 6), (12, 13), (1, 300)])
def test_hidden_positions(window, low):
    """Half of the positions hidden; then all but one step to the right, which leaves some queries nothing to see."""
    g = torch.Generator(device=DEV).manual_seed(1)
    heads, d, n_win = 3, 32, 2
    qkv, table, _, d_o = make(n_win, window, heads, d, g)
    table[torch.rand(len(table), generator=g, device=DEV) < 0.5] = low
    _, _, _, dtable = run_both(qkv, table, None, d_o, n_win, window, heads, d)
    assert not dtable[table <= PB.HIDDEN].any()
    only = torch.full_like(table, low)
    h, w = window
    only[(h - 1) * (2 * w - 1) + (w - 1) - 1] = 0.3           # x_i - x_j = -1: the key one to the right
    o, lse, dqkv, dtable = run_both(qkv, only, None, d_o, n_win, window, heads, d)
    last = torch.arange(h * w, device=DEV) % w == w - 1       # nothing there
    blind = last.repeat(n_win)
    assert not o[blind].any() and o[~blind].any() and bool(lse[:, :, last].isinf().all())
    assert not dqkv[blind][:, :heads * d].any()
    # one key each: a probability of one, whatever the scores
    right = torch.roll(qkv[:, 2 * heads * d:], -1, 0)
    assert torch.equal(o[~blind], right[~blind])
    everything = torch.full_like(table, low)
    o, lse, dqkv, dtable = run_both(qkv, everything, None, d_o, n_win, window, heads, d)
    assert not o.any() and not dqkv.any() and not dtable.any()


def test_head_that_sees_nothing_beside_others():
    g = torch.Generator(device=DEV).manual_seed(2)
    qkv, table, buckets, d_o = make(2, (9, 20), 3, 64, g, 4)
    table[:, 1] = -math.inf
    o, *_ = run_both(qkv, table, buckets, d_o, 2, (9, 20), 3, 64)
    assert not o[:, 64:128].any() and o[:, :64].any()


def test_far_scores_and_biases():
    g = torch.Generator(device=DEV).manual_seed(3)
    for strength, scale in ((30.0, None), (1.0, 2.0), (1.0, 0.0), (3.0, -0.3), (1000.0, None)):
        qkv, table, _, d_o = make(2, (10, 16), 2, 64, g, strength=strength)
        run_both(qkv, table, None, d_o, 2, (10, 16), 2, 64, scale)


@pytest.mark.parametrize("d", [20, 64, 12, 1, 100])
@pytest.mark.parametrize("gap", [0, 8, 3])
def test_pitches_and_odd_heads(d, gap):
    g = torch.Generator(device=DEV).manual_seed(d + gap)
    heads, n_win, window = 3, 2, (7, 11)
    n = 77
    qkv, table, _, d_o = make(n_win, window, heads, d, g)
    wide = torch.zeros((n_win * n, 3 * heads * d + gap), device=DEV, dtype=BF)
    wide[:, :3 * heads * d] = qkv
    qkv = wide[:, :3 * heads * d]
    out = torch.full((n_win * n, heads * d + gap), 4.0, device=DEV, dtype=BF)
    place = torch.full((n_win * n, 3 * heads * d + gap), 4.0, device=DEV, dtype=BF)
    sums = torch.full(table.shape, 0.25, device=DEV)
    f = formula(qkv, window, heads, d, table, None, 1 / math.sqrt(d))
    lse = torch.empty((n_win, heads, n), device=DEV)
    o, lse2 = PB.biased_attn_fwd(qkv, n_win, window, heads, d, table, out=out[:, :heads * d], lse=lse)
    assert lse2 is lse and o.data_ptr() == out.data_ptr()
    forward_check(o, lse, f)
    dqkv, dtable = PB.biased_attn_bwd(d_o, qkv, o, lse, n_win, window, heads, d, table, dqkv=place[:, :3 * heads * d], dtable=sums)
    assert dtable is sums and dqkv.data_ptr() == place.data_ptr()
    backward_check(d_o, o, dqkv, dtable, f, window, heads, d, 1 / math.sqrt(d), table.shape[0], base=0.25)
    if gap:
        assert bool((out[:, heads * d:] == 4).all()) and bool((place[:, 3 * heads * d:] == 4).all())
    none, t = PB.biased_attn_bwd(d_o, qkv, o, lse, n_win, window, heads, d, table, need_dtable=False)
    assert t is None and torch.equal(none, dqkv)


def test_sums_added_to_with_buckets_and_one_token():
    g = torch.Generator(device=DEV).manual_seed(5)
    for n_win, window, rows in ((3, (6, 7), 9), (4, (1, 1), None)):
        qkv, table, buckets, d_o = make(n_win, window, 2, 32, g, rows)
        o, lse = PB.biased_attn_fwd(qkv, n_win, window, 2, 32, table, buckets)
        args = (d_o, qkv, o, lse, n_win, window, 2, 32, table, buckets)
        alone = PB.biased_attn_bwd(*args)[1]
        sums = torch.full(table.shape, 3.0, device=DEV)
        PB.biased_attn_bwd(*args, dtable=sums)
        assert torch.equal(sums, 3.0 + alone)
    assert not alone.any()        # one token sees itself whatever the bias


def test_no_windows():
    table = torch.zeros((PB.relative_positions((3, 4)), 2), device=DEV)
    qkv = torch.empty((0, 3 * 2 * 32), device=DEV, dtype=BF)
    o, lse = PB.biased_attn_fwd(qkv, 0, (3, 4), 2, 32, table)
    assert o.shape == (0, 64) and lse.shape == (0, 2, 12)
    dqkv, dtable = PB.biased_attn_bwd(o, qkv, o, lse, 0, (3, 4), 2, 32, table)
    assert dqkv.shape == qkv.shape and not dtable.any()


def test_bucket_outside_the_table_is_recorded():
    from aeris_gb_b200.ops import lib as _l
    g = torch.Generator(device=DEV).manual_seed(6)
    for bad in (-1, 5, 2 ** 40):
        qkv, table, buckets, _ = make(2, (5, 6), 2, 32, g, 5)
        buckets = buckets.long()
        buckets[7] = bad
        PB.biased_attn_fwd(qkv, 2, (5, 6), 2, 32, table, buckets)
        with pytest.raises(_l.KernelError, match="bounds"):
            _l.check_status()


def test_many_windows_and_many_heads():
    """More slices and groups of heads than one (sums over 2,000 windows; matrices of 1,600 tokens)."""
    g = torch.Generator(device=DEV).manual_seed(7)
    run_both(*make(2000, (4, 4), 2, 16, g), 2000, (4, 4), 2, 16)
    run_both(*make(1, (40, 40), 30, 16, g), 1, (40, 40), 30, 16)


@pytest.mark.parametrize("n_win,window,heads,d", [(40, (8, 8), 24, 64), (30, (8, 8), 24, 128), (60, (3, 3), 40, 16), (20, (12, 12), 24, 32),
                                                  (20, (9, 11), 24, 72), (25, (16, 20), 9, 64), (30, (13, 20), 10, 128), (10, (30, 30), 5, 64),
                                                  (2, (8, 8), 300, 64), (1, (16, 17), 200, 32), (1, (20, 13), 160, 128), (6, (40, 40), 7, 64)])
def test_several_heads_in_the_run_of_a_block(n_win, window, heads, d):
    """More items than multiprocessors: blocks go from the table of one head to that of the next."""
    g = torch.Generator(device=DEV).manual_seed(n_win)
    run_both(*make(n_win, window, heads, d, g), n_win, window, heads, d)


@pytest.mark.parametrize("n_win,window,heads,d", [(700, (17, 4), 1, 72), (900, (3, 20), 1, 64), (149, (8, 16), 2, 32), (40, (12, 12), 17, 64),
                                                  (40, (10, 13), 3, 128), (90, (12, 17), 1, 96), (20, (16, 16), 9, 72), (19, (1, 257), 5, 128),
                                                  (17, (20, 20), 33, 80)])
def test_few_tiles_of_many_windows(n_win, window, heads, d):
    g = torch.Generator(device=DEV).manual_seed(n_win)
    run_both(*make(n_win, window, heads, d, g), n_win, window, heads, d)


def test_same_bits_captured_and_on_another_stream():
    g = torch.Generator(device=DEV).manual_seed(8)
    qkv, table, buckets, d_o = make(20, (9, 16), 4, 64, g, 50)

    def both():
        o, lse = PB.biased_attn_fwd(qkv, 20, (9, 16), 4, 64, table, buckets)
        return (o, lse, *PB.biased_attn_bwd(d_o, qkv, o, lse, 20, (9, 16), 4, 64, table, buckets))

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


def test_table_gradient_against_differences():
    """Sum of dO * o for a moved entry of the table: o is rounded to bf16, so the step is large and the bound says so."""
    g = torch.Generator(device=DEV).manual_seed(9)
    qkv, table, buckets, d_o = make(40, (6, 6), 2, 32, g, 6)
    o, lse = PB.biased_attn_fwd(qkv, 40, (6, 6), 2, 32, table, buckets)
    _, dtable = PB.biased_attn_bwd(d_o, qkv, o, lse, 40, (6, 6), 2, 32, table, buckets)
    h = 2.0 ** -3
    for b in range(6):
        for head in range(2):
            moved = [table.clone() for _ in range(2)]
            moved[0][b, head] += h
            moved[1][b, head] -= h
            up, down = (PB.biased_attn_fwd(qkv, 40, (6, 6), 2, 32, t, buckets)[0].double() for t in moved)
            do = d_o.double()
            slope = float((do * (up - down)).sum() / (2 * h))
            # P and o rounded to bf16 twice each, independently of one another (4 deviations of their root mean square), and
            # a third derivative of at most a sixteenth of the terms
            noise = 4 * HALF * float((do * up).square().sum().sqrt() * 2) / (2 * h)
            size = float((do.abs() * up.abs()).sum())
            assert abs(slope - float(dtable[b, head])) < noise + h * h / 16 * size / 6


@pytest.mark.parametrize("window", [(8, 8), (10, 13)])
def test_offsets_past_32_bits(window):
    """Rows of one large matrix (8.6 GB) whose last ones are further than 2^32 elements from the first: the same bits as of rows that
    are close together."""
    n, heads, d = window[0] * window[1], 2, 24
    n_win = 4096 // n
    g = torch.Generator(device=DEV).manual_seed(2)
    qkv, table, _, d_o = make(n_win, window, heads, d, g)
    rows, inner = n_win * n, heads * d
    wide = torch.empty((rows, (2 ** 32 // rows + 4096) // 8 * 8), device=DEV, dtype=BF)
    assert (rows - 1) * wide.stride(0) > 2 ** 32
    far = [wide[:, 8 + 256 * i:8 + 256 * i + k * inner] for i, k in enumerate((3, 1, 1, 3))]
    far[0].copy_(qkv)
    far[1].copy_(d_o)
    want, lse = PB.biased_attn_fwd(qkv, n_win, window, heads, d, table)
    o, again = PB.biased_attn_fwd(far[0], n_win, window, heads, d, table, out=far[2])
    assert torch.equal(o, want) and torch.equal(again, lse)
    grad, dtable = PB.biased_attn_bwd(d_o, qkv, want, lse, n_win, window, heads, d, table)
    g2, dt2 = PB.biased_attn_bwd(far[1], far[0], o, lse, n_win, window, heads, d, table, dqkv=far[3])
    assert torch.equal(g2, grad) and torch.equal(dt2, dtable)


@pytest.mark.parametrize("window,heads,d", [((4, 4), 2, 32), ((7, 7), 3, 64), ((9, 10), 2, 24), ((12, 12), 3, 40), ((20, 20), 2, 64), ((12, 12), 2, 128)])
def test_two_calls_at_once(window, heads, d):
    """Other data on two streams, eight times beside one another: the bits of calls by themselves."""
    n_win, sets = 30, []
    for i in range(2):
        g = torch.Generator(device=DEV).manual_seed(i)
        sets.append(make(n_win, window, heads, d, g))

    def both(qkv, table, _, d_o):
        o, lse = PB.biased_attn_fwd(qkv, n_win, window, heads, d, table)
        return o, lse, *PB.biased_attn_bwd(d_o, qkv, o, lse, n_win, window, heads, d, table)

    want = [both(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(8):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(both(*s))
    torch.cuda.synchronize()
    for i, results in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(results, want[i % 2]))


@pytest.mark.parametrize("n_win,window,heads,d", [(2, (5, 6), 2, 32), (2, (9, 13), 2, 64), (2, (12, 16), 3, 64), (3, (10, 16), 2, 128), (1, (20, 20), 5, 72)])
def test_bucket_outside_the_table_ends_every_kernel_of_the_call(n_win, window, heads, d):
    """Recorded in both directions, and soon: no kernel of the backward pass waits for what another has left undone (limits of
    waits are 2 s). Later calls are as before."""
    from aeris_gb_b200.ops import lib as _l
    g = torch.Generator(device=DEV).manual_seed(6)
    qkv, table, buckets, d_o = make(n_win, window, heads, d, g, 5)

    def both(b):
        o, lse = PB.biased_attn_fwd(qkv, n_win, window, heads, d, table, b)
        return o, lse, *PB.biased_attn_bwd(d_o, qkv, o, lse, n_win, window, heads, d, table, b)

    want = both(buckets)
    bad = buckets.clone()
    bad[7] = 5
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for call in (lambda: PB.biased_attn_fwd(qkv, n_win, window, heads, d, table, bad),
                 lambda: PB.biased_attn_bwd(d_o, qkv, want[0], want[1], n_win, window, heads, d, table, bad)):
        start.record()
        call()
        end.record()
        with pytest.raises(_l.KernelError, match="bounds"):
            _l.check_status()
        assert start.elapsed_time(end) < 1000
    assert all(map(torch.equal, both(buckets), want))


@pytest.mark.parametrize("window", [(3, 5), (10, 11)])
@pytest.mark.parametrize("heads,d", [(5, 1), (1, 1), (1, 5), (1, 20), (2, 7)])
def test_results_of_padded_heads_go_on_into_the_backward_pass(heads, d, window):
    g = torch.Generator(device=DEV).manual_seed(heads + d)
    o, _, dqkv, _ = run_both(*make(3, window, heads, d, g), 3, window, heads, d)
    assert o.is_contiguous() and dqkv.is_contiguous()


@pytest.mark.parametrize("heads,d", [(1, 20), (3, 1), (1, 1), (2, 20)])
def test_plain_attention_of_padded_heads_goes_on_into_its_backward_pass(heads, d):
    """The same by the kernels without a bias, whose backward pass takes o and its gradient in rows of one pitch."""
    g = torch.Generator(device=DEV).manual_seed(heads + d)
    n_win, window = 3, (10, 13)
    qkv, table, _, d_o = make(n_win, window, heads, d, g)
    o, lse = A.attn_fwd(qkv, n_win, 130, heads, d)
    dqkv = A.attn_bwd(qkv, o, d_o, lse, n_win, 130, heads, d)
    f = formula(qkv, window, heads, d, 0 * table, None, 1 / math.sqrt(d))
    forward_check(o, lse, f)
    backward_check(d_o, o, dqkv, None, f, window, heads, d, 1 / math.sqrt(d), len(table))


@pytest.mark.parametrize("window,heads,d", [((95, 95), 1, 64), ((1, 9000), 1, 40), ((9001, 1), 1, 128), ((1, 15700), 1, 64), ((126, 125), 1, 128)])
def test_windows_whose_tables_do_not_fit_beside_the_tiles(window, heads, d):
    """Slices of a head's table, and beyond them (15,000 tokens and more) the table in memory."""
    g = torch.Generator(device=DEV).manual_seed(window[0])
    run_both(*make(1, window, heads, d, g), 1, window, heads, d)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("window,heads,d", [((3, 5), 2, 24), ((9, 13), 3, 40), ((12, 13), 2, 128), ((17, 19), 2, 64), ((5, 7), 1, 20)])
@pytest.mark.parametrize("gap", [8, 3])
def test_what_lies_between_rows_is_not_read_into_results(window, heads, d, gap):
    g = torch.Generator(device=DEV).manual_seed(d + gap)
    n_win, n = 3, window[0] * window[1]
    tight = make(n_win, window, heads, d, g)
    qkv, d_o = (torch.full((t.shape[0] + 1, t.shape[1] + gap), math.nan, device=DEV, dtype=BF)[:-1, :t.shape[1]] for t in (tight[0], tight[3]))
    qkv.copy_(tight[0])
    d_o.copy_(tight[3])
    assert n_win * n == len(qkv)
    run_both(qkv, tight[1], None, d_o, n_win, window, heads, d)
