"""Refusals of the norms of queries and keys: made on the host, before anything is launched."""
import pytest
import torch

from aeris_gb_b200.ops import qk_norm as QN

ROWS, H, HK, D, L = 6, 4, 2, 16, 3


def args(**over):
    a = dict(q=torch.randn(ROWS, H, D), k=torch.randn(ROWS, HK, D), wq=torch.ones(D), wk=torch.ones(D),
             cos=torch.ones(L, D // 2), sin=torch.zeros(L, D // 2), positions=None, q_out=None, k_out=None)
    a.update(over)
    return a


def forward(a):
    return QN.qk_norm_fwd(a["q"], a["k"], a["wq"], a["wk"], a["cos"], a["sin"], eps=1e-6, positions=a["positions"],
                          q_out=a["q_out"], k_out=a["k_out"])


BAD = {
    "rows differ": dict(k=torch.randn(ROWS + 1, HK, D)),
    "widths differ": dict(k=torch.randn(ROWS, HK, D + 2)),
    "two dimensions": dict(q=torch.randn(ROWS, H * D)),
    "odd width": dict(q=torch.randn(ROWS, H, 15), k=torch.randn(ROWS, HK, 15)),
    "too wide": dict(q=torch.randn(ROWS, H, 258), k=torch.randn(ROWS, HK, 258)),
    "no heads": dict(k=torch.randn(ROWS, 0, D)),
    "half": dict(q=torch.randn(ROWS, H, D).half(), k=torch.randn(ROWS, HK, D).half()),
    "types differ": dict(k=torch.randn(ROWS, HK, D).bfloat16()),
    "channels apart": dict(q=torch.randn(ROWS, D, H).transpose(1, 2)),
    "weight of another width": dict(wq=torch.ones(D + 2)),
    "weight types differ": dict(wk=torch.ones(D).bfloat16()),
    "weight with gaps": dict(wk=torch.ones(2 * D)[::2]),
    "sin without cos": dict(cos=None),
    "positions without angles": dict(cos=None, sin=None, positions=torch.zeros(ROWS, dtype=torch.int32)),
    "angles in bf16": dict(cos=torch.ones(L, D // 2).bfloat16(), sin=torch.ones(L, D // 2).bfloat16()),
    "more angles than pairs": dict(cos=torch.ones(L, D), sin=torch.ones(L, D)),
    "angles of unlike length": dict(sin=torch.ones(L + 1, D // 2)),
    "empty table": dict(cos=torch.ones(0, D // 2), sin=torch.ones(0, D // 2)),
    "positions of another length": dict(positions=torch.zeros(ROWS + 1, dtype=torch.int32)),
    "positions in floating point": dict(positions=torch.zeros(ROWS)),
    "positions with gaps": dict(positions=torch.zeros(2 * ROWS, dtype=torch.int64)[::2]),
    "result of another shape": dict(q_out=torch.empty(ROWS, H + 1, D)),
    "result of another type": dict(k_out=torch.empty(ROWS, HK, D).bfloat16()),
    "expanded result": dict(q_out=torch.empty(1, H, D).expand(ROWS, H, D)),
    "result with overlapping heads": dict(q_out=torch.empty(ROWS * H * D).as_strided((ROWS, H, D), (H * D, D // 2, 1))),
}


@pytest.mark.parametrize("what", BAD)
def test_refused(what):
    with pytest.raises(ValueError):
        forward(args(**BAD[what]))


def test_cpu_tensors_are_refused_and_not_computed_elsewhere():
    with pytest.raises(ValueError, match="GPU"):
        forward(args())


def test_results_in_one_place_are_refused():
    t = torch.empty(ROWS, H, D)
    with pytest.raises(ValueError, match="same memory"):
        forward(args(q_out=t, k_out=t[:, :HK]))


@pytest.mark.parametrize("bad", [dict(dq=torch.randn(ROWS, H, D + 2)), dict(dk=torch.randn(ROWS, HK, D).bfloat16()),
                                 dict(dwq=torch.zeros(D)), dict(dwq=torch.zeros(D), dwk=torch.zeros(D + 1)),
                                 dict(dwq=torch.zeros(D), dwk=torch.zeros(D).bfloat16()),
                                 dict(zip(("dwq", "dwk"), (lambda t: (t[:D], t[4:D + 4]))(torch.zeros(2 * D)))),
                                 dict(dq_out=torch.empty(ROWS, 1, D).expand(ROWS, H, D))])
def test_backward_refuses(bad):
    a = args()
    g = dict(dq=torch.randn(ROWS, H, D), dk=torch.randn(ROWS, HK, D), dwq=None, dwk=None, dq_out=None)
    g.update(bad)
    with pytest.raises(ValueError):
        QN.qk_norm_bwd(g["dq"], g["dk"], a["q"], a["k"], a["wq"], a["wk"], a["cos"], a["sin"], eps=1e-6, dwq=g["dwq"],
                       dwk=g["dwk"], dq_out=g["dq_out"])


@pytest.mark.parametrize("shape,strides,fine", [((5, 3, 8), (24, 8, 1), True), ((5, 3, 8), (8, 40, 1), True),
                                                ((5, 3, 8), (100, 8, 1), True), ((1, 3, 8), (0, 8, 1), True),
                                                ((5, 1, 8), (8, 0, 1), True), ((5, 3, 8), (20, 8, 1), False),
                                                ((5, 3, 8), (0, 8, 1), False), ((5, 3, 8), (8, 36, 1), False)])
def test_overlap_of_results(shape, strides, fine):
    t = torch.empty(1000).as_strided(shape, strides)
    assert QN._apart(t) == fine


def sections(pitch, q_at, k_at):
    """q [ROWS, H, D] and k [ROWS, HK, D] out of one matrix's rows, from those elements of a row on."""
    m = torch.zeros(ROWS, pitch)
    return m[:, q_at:q_at + H * D].unflatten(1, (H, D)), m[:, k_at:k_at + HK * D].unflatten(1, (HK, D))


def placements():
    """(whether the call is taken, q, k, q_out, k_out)"""
    q, k = torch.randn(ROWS, H, D), torch.randn(ROWS, HK, D)
    s, t = sections((H + HK) * D, 0, H * D), sections((H + HK) * D, 0, (H - 1) * D)
    one = torch.zeros(ROWS, 2, HK, 3, D)                  # q, k and v of every head side by side, of two groups of heads
    first, second = one[:, 0, :, 0], one[:, 0, :, 1]
    long = torch.randn((ROWS + 1) * H * D)
    rows = long[:-H * D].view(ROWS, H, D)
    back = torch.zeros(H, ROWS, D).transpose(0, 1)        # rows inside heads
    return {
        "sections": (True, q, k, *s),
        "in place": (True, q, k, q, k),
        "sections in place": (True, *s, *s),
        "q alone in place": (True, *s, s[0], None),
        "head by head": (True, q[:, :HK], k, first, second),
        "head by head in place": (True, first, second, first, second),
        "rows inside heads, in place": (True, back, k, back, k),
        "q over k": (False, q, q[:, :HK], q, None),
        "k over q": (False, q, k, None, q[:, :HK]),
        "k over q's last heads": (False, q, k, None, q[:, H - HK:]),
        "q and k changed over": (False, first, second, second, first),
        "results over each other": (False, q, k, *t),
        "results in one place": (False, q[:, :HK], k, first, first),
        "a row behind the input": (False, rows, k, long[H * D:].view(ROWS, H, D), None),
        "a channel behind the input": (False, rows, k, long[1:1 + ROWS * H * D].view(ROWS, H, D), None),
        "over the input in another order": (False, rows, k, long[:-H * D].view(H, ROWS, D).transpose(0, 1), None),
    }


@pytest.mark.parametrize("what", placements())
def test_results_over_another_one_s_elements_are_refused(what):
    """Blocks of q and blocks of k run at the same time. What is taken here goes on to ask for a GPU."""
    fine, q, k, q_out, k_out = placements()[what]
    with pytest.raises(ValueError) as e:
        forward(args(q=q, k=k, q_out=q_out, k_out=k_out))
    assert ("on a GPU" in str(e.value)) == fine, e.value
    a = args()
    # the gradients of q and k over those of the results
    with pytest.raises(ValueError) as e:
        QN.qk_norm_bwd(q, k, torch.randn(q.shape), torch.randn(k.shape), a["wq"], a["wk"], a["cos"], a["sin"], eps=1e-6,
                       dq_out=q_out, dk_out=k_out)
    assert ("on a GPU" in str(e.value)) == fine, e.value
    # and over the inputs themselves
    with pytest.raises(ValueError) as e:
        QN.qk_norm_bwd(torch.randn(q.shape), torch.randn(k.shape), q, k, a["wq"], a["wk"], a["cos"], a["sin"], eps=1e-6,
                       dq_out=q_out, dk_out=k_out)
    assert ("on a GPU" in str(e.value)) == fine, e.value


def test_shared_memory_against_every_byte():
    """What is said to be apart is apart; sections and whole tensors are told apart exactly."""
    import random
    from aeris_gb_b200.ops import lib as L
    rnd, base = random.Random(1), torch.empty(400, dtype=torch.uint8)

    def one(d, rows):
        heads = rnd.randint(1, 3)
        head = d * rnd.choice([1, 1, 1, 2, 0])
        return base.as_strided((rows, heads, d), (rnd.choice([heads * head, 24, 24, d, 0]), head, 1), rnd.randint(0, 60))

    def places(t):
        (r, h, d), (a, b, _), o = t.shape, t.stride(), t.storage_offset()
        return {o + i * a + j * b + k for i in range(r) for j in range(h) for k in range(d)}

    met = exact = 0
    for _ in range(20000):
        d, rows = rnd.choice([2, 4, 6]), rnd.randint(1, 4)
        a, b = one(d, rows), one(d, rows)
        want, got = bool(places(a) & places(b)), L.share_memory(a, b)
        met += want
        assert got or not want
        if rows > 1 and a.stride(0) == b.stride(0) == 24 and all(t.shape[1] == 1 or t.stride(1) == d for t in (a, b)):
            assert got == want
            exact += 1
        wa, wb = ((t, t.data_ptr(), *t.stride()[:2], t.shape[1]) for t in (a, b))
        assert QN._share(wa, wb, rows, d, 1) == got
    assert 1000 < met < 19000 and exact > 100
