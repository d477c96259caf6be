"""Window attention with a position bias in windows of up to 96 tokens, against its formulas in 64 bits (tolerances: see the tests of
larger windows)."""
import pytest
import torch

import test_position_bias_gpu as T
from aeris_gb_b200.ops import position_bias as PB

pytestmark = pytest.mark.gpu
DEV = T.DEV


@pytest.mark.parametrize("d", [8, 16, 24, 64, 72, 128])
@pytest.mark.parametrize("window", [(1, 1), (1, 2), (3, 1), (4, 4), (1, 16), (17, 1), (3, 7), (4, 8), (3, 11), (6, 8), (7, 7), (1, 63), (8, 8), (64, 1), (5, 13), (8, 10), (1, 81),
                                    (8, 12), (96, 1)])
def test_sizes(window, d):
    for n_win, heads in ((1, 1), (5, 3), (70, 2)):
        g = torch.Generator(device=DEV).manual_seed(n_win + d)
        T.run_both(*T.make(n_win, window, heads, d, g), n_win, window, heads, d)


@pytest.mark.parametrize("n_win,window,heads,d", [(2000, (4, 4), 3, 32), (1500, (7, 7), 2, 64), (900, (5, 6), 5, 16), (3, (8, 8), 700, 8),
                                                  (701, (6, 8), 1, 40), (700, (17, 4), 1, 72), (400, (9, 10), 2, 64)])
def test_many_windows_and_many_heads(n_win, window, heads, d):
    g = torch.Generator(device=DEV).manual_seed(n_win)
    T.run_both(*T.make(n_win, window, heads, d, g), n_win, window, heads, d)


@pytest.mark.parametrize("window", [(4, 4), (5, 5), (6, 7), (7, 8), (9, 8), (9, 10)])
def test_values_that_are_not_finite_stay_in_their_window_and_head(window):
    n, heads, d, n_win = window[0] * window[1], 2, 24, 11
    g = torch.Generator(device=DEV).manual_seed(3)
    qkv, table, _, d_o = T.make(n_win, window, heads, d, g)
    o, lse = PB.biased_attn_fwd(qkv, n_win, window, heads, d, table)
    grad, _ = PB.biased_attn_bwd(d_o, qkv, o, lse, n_win, window, heads, d, table)
    bad, bad_do = qkv.clone(), d_o.clone()
    for part, (win, value) in enumerate(((2, float("inf")), (4, float("nan")), (6, float("-inf")))):
        bad[win * n:(win + 1) * n, part * heads * d:part * heads * d + d] = value       # head 0
    bad_do[8 * n:9 * n, :d] = float("nan")
    ob, lb = PB.biased_attn_fwd(bad, n_win, window, heads, d, table)
    gb, _ = PB.biased_attn_bwd(bad_do, bad, ob, lb, n_win, window, heads, d, table, need_dtable=False)
    clean = [w for w in range(n_win) if w not in (2, 4, 6, 8)]
    by = lambda t, k: t.reshape(n_win, n, k, heads, d)      # noqa: E731
    assert torch.equal(by(ob, 1)[clean], by(o, 1)[clean]) and torch.equal(by(ob, 1)[..., 1, :], by(o, 1)[..., 1, :])
    assert torch.equal(by(gb, 3)[clean], by(grad, 3)[clean]) and torch.equal(by(gb, 3)[..., 1, :], by(grad, 3)[..., 1, :])
    assert torch.equal(lb[clean], lse[clean]) and torch.equal(lb[:, 1], lse[:, 1])
    assert by(gb, 3)[8, :, :2, 0].isnan().all()


def test_rows_outside_stay():
    """Results between other columns and before other rows: what is beside them is left."""
    n_win, window, heads, d = 7, (5, 7), 2, 32
    n, inner = 35, 64
    g = torch.Generator(device=DEV).manual_seed(5)
    qkv, table, _, d_o = T.make(n_win, window, heads, d, g)
    rows = n_win * n
    wide = torch.full((rows + 3, inner + 16), 7.0, device=DEV, dtype=T.BF)
    wide3 = torch.full((rows + 3, 3 * inner + 16), 7.0, device=DEV, dtype=T.BF)
    o, lse = PB.biased_attn_fwd(qkv, n_win, window, heads, d, table, out=wide[:rows, 8:8 + inner])
    want, _ = PB.biased_attn_fwd(qkv, n_win, window, heads, d, table)
    assert torch.equal(o, want)
    PB.biased_attn_bwd(d_o, qkv, want, lse, n_win, window, heads, d, table, dqkv=wide3[:rows, 8:8 + 3 * inner])
    grad, _ = PB.biased_attn_bwd(d_o, qkv, want, lse, n_win, window, heads, d, table)
    assert torch.equal(wide3[:rows, 8:8 + 3 * inner], grad)
    for t, k in ((wide, inner), (wide3, 3 * inner)):
        assert bool((t[rows:] == 7).all() and (t[:, :8] == 7).all() and (t[:, 8 + k:] == 7).all())


def test_same_bits_in_two_graphs_beside_one_another():
    shapes = [(300, (7, 7), 3, 32), (200, (4, 4), 4, 64)]
    sets = []
    for s in shapes:
        g = torch.Generator(device=DEV).manual_seed(s[0])
        sets.append((s, *T.make(s[0], s[1], s[2], s[3], g, 9)))

    def both(s, qkv, table, buckets, d_o):
        o, lse = PB.biased_attn_fwd(qkv, *s, table, buckets)
        return o, lse, *PB.biased_attn_bwd(d_o, qkv, o, lse, *s, table, buckets)

    want = [both(*s) for s in sets]
    torch.cuda.synchronize()
    graphs, held = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(both(*s))
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, held):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
