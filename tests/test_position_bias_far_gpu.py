"""Window attention with biases far from zero in windows whose tokens are no multiple of 16, against its formulas in 64 bits
(tolerances: see the tests of other windows). The last tile then has rows of zeros behind the window's, which a bias of any size leaves
without weight.

The table's gradient takes pairs whose bias is within 64 in log2 units as 2^(score - lse) times 2^bias, the bias left out of the
score; fp32 ends at 2^-126, so that a probability below 2^-62 may be lost: 2^-62 |dp - delta| more of every such pair.
"""
import math

import pytest
import torch

import test_position_bias_gpu as T
from aeris_gb_b200.ops import position_bias as PB

pytestmark = pytest.mark.gpu
DEV = T.DEV


def table_check(d_o, dtable, table, f, n, heads, d):
    """As the other windows' tests, and what may be lost."""
    _, _, v, p, _, es, index = f
    do = T.heads_of(d_o, n, heads, d)[0]
    dp, dp_size = do @ v.transpose(-1, -2), do.abs() @ v.abs().transpose(-1, -2)
    rest = dp - (p * dp).sum(-1, keepdim=True)
    ds, e_p, e_dp = p * rest, 2 * es * p, (d / 16 + 4) * 2.0 ** -23 * dp_size
    e_delta = (p * e_dp + e_p * rest.abs()).sum(-1, keepdim=True) + (n / 16 + 16) * 2.0 ** -23 * (p * dp_size).sum(-1, keepdim=True)
    lost = 2.0 ** -62 * (table.double().T[:, index].abs() * T.LOG2E <= 65) * (rest.abs() + e_dp + e_delta)
    e_ds = e_p * rest.abs() + p * (e_dp + e_delta) + 2.0 ** -22 * ds.abs() + lost
    zero = torch.zeros(table.shape, dtype=torch.float64, device=DEV)
    add = lambda x: zero.index_add(0, index.reshape(-1), x.sum(0).flatten(1).T)  # noqa: E731
    want = add(ds)
    T.within(dtable, want, add(e_ds + (ds.shape[0] + n / 8 + 64) * 2.0 ** -24 * ds.abs()) + 2.0 ** -23 * want.abs())


@pytest.mark.parametrize("window,heads,d", [((9, 13), 2, 64), ((10, 13), 1, 128), ((12, 13), 3, 40), ((13, 17), 2, 64), ((13, 17), 2, 128),
                                            ((1, 97), 2, 72), ((30, 30), 2, 64), ((30, 30), 1, 128)])
@pytest.mark.parametrize("strength,shift", [(30.0, 0.0), (1000.0, 0.0), (1.0, 100.0), (1.0, -100.0)])
def test_far_biases_where_tiles_reach_past_the_window(window, heads, d, strength, shift):
    g = torch.Generator(device=DEV).manual_seed(window[1] + d)
    n, n_win = window[0] * window[1], 3
    qkv, table, _, d_o = T.make(n_win, window, heads, d, g, strength=strength)
    table = table + shift
    o, lse = PB.biased_attn_fwd(qkv, n_win, window, heads, d, table)
    dqkv, dtable = PB.biased_attn_bwd(d_o, qkv, o, lse, n_win, window, heads, d, table)
    assert all(bool(t.isfinite().all()) for t in (o, lse, dqkv, dtable))
    f = T.formula(qkv, window, heads, d, table, None, 1 / math.sqrt(d))
    T.forward_check(o, lse, f)
    T.backward_check(d_o, o, dqkv, None, f, window, heads, d, 1 / math.sqrt(d), len(table))
    table_check(d_o, dtable, table, f, n, heads, d)
