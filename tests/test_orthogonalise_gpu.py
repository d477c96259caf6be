"""Orthogonalisation of matrices, and the optimizer step on it, against their formulas in 64 bits.

Tolerance of an orthogonalised matrix: the kernels keep X and the square factors in fp16 and sum in fp32, so what they are off by
is the roundings of the stored arrays, amplified by the steps that follow. :func:`model` runs the formula in 64 bits twice,
plainly and with every stored array multiplied by 1 + delta, delta drawn evenly from a half step (2^-11) to either side: larger
than roundings are on average. Twice the largest distance of eight such draws (the few roundings of a matrix of one row can
cancel in a single one: 7e-5 to 3e-3 for one element), and the rounding of the bf16 result (half a step, 2^-8 of each value), is
allowed for; single elements may be off by six times the root mean square of that.
"""
import math

import pytest
import torch

from aeris_gb_b200.ops import lib as _l
from aeris_gb_b200.ops import orthogonalise as OR

pytestmark = pytest.mark.gpu
DEV = "cuda"
A, B, C = OR.COEFFICIENTS
U32 = 2.0 ** -24


def noisy(x, g, scale):
    if g is None:
        return x
    delta = (2 * torch.rand(x.shape, generator=g, device=DEV, dtype=torch.float64) - 1)
    return x * (1 + delta * 2.0 ** -11) + delta * 2.0 ** -25 / scale          # the second: steps below fp16's normal range


def iterate(x, steps, eps, g=None):
    if x.shape[-2] > x.shape[-1]:
        return iterate(x.mT, steps, eps, g).mT
    x = noisy(x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(eps), g, 512)
    for _ in range(steps):
        s = noisy(x @ x.mT, g, 512)
        one = torch.eye(x.shape[-2], dtype=torch.float64, device=DEV)
        x = noisy(noisy(A * one + B * s + C * (s @ s), g, 512) @ x, g, 512)
    return x


def model(x, steps=5, eps=1e-7):
    """(exact result, 2-norm that each matrix may be off by before its last rounding)."""
    x = x.double()
    want = iterate(x, steps, eps)
    off = [(iterate(x, steps, eps, torch.Generator(device=DEV).manual_seed(k)) - want).square().sum((-2, -1), keepdim=True).sqrt()
           for k in range(8)]
    return want, 2 * torch.stack(off).amax(0)


def close(got, want, off, last=2.0 ** -8):
    got = got.double()
    n = want.shape[-2] * want.shape[-1]
    d = got - want
    assert bool((d.square().sum((-2, -1), keepdim=True).sqrt() <= off + last * want.square().sum((-2, -1), keepdim=True).sqrt()).all())
    assert bool((d.abs() <= last * want.abs() + 6 * off / math.sqrt(n) + 1e-30).all())


def gradient(*shape, noise=0.5, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = min(shape[-2:])
    s = torch.arange(1, r + 1, device=DEV).float().rsqrt()
    x = (torch.randn((*shape[:-1], r), generator=g, device=DEV) * s) @ torch.randn((*shape[:-2], r, shape[-1]), generator=g, device=DEV)
    return x / x.square().mean().sqrt() + noise * torch.randn(shape, generator=g, device=DEV)


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (3, 200), (200, 3), (31, 33), (63, 65), (64, 64), (65, 64), (128, 128), (128, 129), (129, 127),
          (127, 640), (192, 192), (256, 256), (257, 300), (300, 257), (384, 1024), (1001, 333), (320, 2000), (515, 515), (768, 640),
          (1, 385), (2, 5000), (64, 4000), (65, 700), (100, 13001), (128, 8192), (5000, 96), (150, 9000), (9001, 300), (512, 5000)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_one_matrix(shape, dt):
    x = gradient(*shape).to(dt)
    close(OR.orthogonalise(x), *model(x))


@pytest.mark.parametrize("count,rows,cols", [(3, 5, 9), (2, 64, 64), (40, 64, 64), (7, 100, 60), (3, 130, 260), (300, 16, 16),
                                             (5, 333, 200), (2, 512, 1536), (9, 384, 384),
                                             (3, 40, 6000), (200, 128, 400), (160, 9, 1000), (3, 1200, 100)])
def test_batches_equal_single_matrices(count, rows, cols):
    x = gradient(count, rows, cols)
    got = OR.orthogonalise(x)
    close(got, *model(x))
    for i in {0, count // 2, count - 1}:
        assert torch.equal(got[i], OR.orthogonalise(x[i]))


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("shape", [(96, 96), (96, 400), (300, 64)])
def test_steps(steps, shape):
    x = gradient(*shape)
    close(OR.orthogonalise(x, steps=steps), *model(x, steps))


@pytest.mark.parametrize("shape", [(200, 200), (150, 600), (100, 900), (60, 90)])
@pytest.mark.parametrize("noise", [0.0, 0.1, 10.0])
def test_spectra(shape, noise):
    x = gradient(*shape, noise=noise)
    close(OR.orthogonalise(x), *model(x))


def test_low_rank():
    g = torch.Generator(device=DEV).manual_seed(3)
    for rank in (1, 4):
        for rows, cols in ((160, 300), (60, 2000), (100, 200)):
            x = torch.randn(rows, rank, generator=g, device=DEV) @ torch.randn(rank, cols, generator=g, device=DEV)
            close(OR.orthogonalise(x), *model(x))


def test_singular_values_end_around_one():
    x = gradient(400, 700)
    s = torch.linalg.svdvals(OR.orthogonalise(x).double())
    assert s.min() > 0.6 and s.max() < 1.25


def test_layouts_of_the_input_and_the_result():
    x = gradient(3, 70, 90)
    want = OR.orthogonalise(x)
    wide = torch.zeros(3, 75, 103, device=DEV)
    for start in (0, 1):                                    # on and off the vectors' grid
        part = wide[:, 2:72, start:start + 90]
        part.copy_(x)
        assert torch.equal(OR.orthogonalise(part), want)
    assert torch.equal(OR.orthogonalise(x.permute(0, 2, 1).contiguous().permute(0, 2, 1)), want)
    assert torch.equal(OR.orthogonalise(x[:1].expand(3, 70, 90)), want[:1].expand(3, 70, 90))
    one = torch.zeros(70 * 90 + 1, device=DEV)[1:].view(70, 90)      # a start off the vectors' grid
    one.copy_(x[1])
    assert torch.equal(OR.orthogonalise(one), want[1])
    low = torch.zeros(70 * 90 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(70, 90)
    low.copy_(x[1])
    assert torch.equal(OR.orthogonalise(low), OR.orthogonalise(low.clone()))
    for pitch, start in ((90, 0), (91, 0), (100, 3), (96, 4)):
        out = torch.full((3, 70, pitch), 7.0, device=DEV, dtype=torch.bfloat16)
        view = out[:, :, start:start + 90]
        assert OR.orthogonalise(x, out=view) is view and torch.equal(view, want)
        assert bool((out[:, :, :start] == 7).all()) and bool((out[:, :, start + 90:] == 7).all())


def test_empty():
    before = _l.launch_count()
    for shape in ((0, 4, 4), (3, 0, 4), (0, 5), (5, 0)):
        assert OR.orthogonalise(torch.empty(shape, device=DEV)).shape == shape
    assert _l.launch_count() == before


def test_zeros_and_values_that_are_no_numbers():
    x = gradient(5, 80, 100)
    want = OR.orthogonalise(x)
    x[1] = 0
    x[2, 3, 4] = float("nan")
    x[3, 0, 0] = float("inf")
    got = OR.orthogonalise(x)
    assert torch.equal(got[0], want[0]) and torch.equal(got[4], want[4]) and bool((got[1] == 0).all())
    assert bool(got[2].isnan().all()) and bool(got[3].isnan().any())


@pytest.mark.parametrize("power", [-60, -30, 30, 60])
def test_scale_of_the_input_does_not_matter(power):
    x = gradient(100, 120)
    assert torch.equal(OR.orthogonalise(x * 2.0 ** power, eps=1e-30), OR.orthogonalise(x))


@pytest.mark.parametrize("shape", [(128, 384), (300, 400), (400, 300), (100, 2000), (33, 1001), (301, 403)], ids=str)
def test_norms_beyond_fp32(shape):
    """Elements up to fp32's largest, whose squares add up to more than it holds: 512 over the norm is below the normal range."""
    x = gradient(*shape).sign() * 2.0 ** 127
    x *= 1 + 0.9 * torch.rand(shape, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    assert bool(x.isfinite().all()) and 512 / x.double().norm() < torch.finfo(torch.float32).tiny
    assert torch.equal(OR.orthogonalise(x), OR.orthogonalise(x * 2.0 ** -100))
    low = x.bfloat16()
    assert torch.equal(OR.orthogonalise(low), OR.orthogonalise(low * 2.0 ** -100))
    assert OR.orthogonalise(x).abs().max() > 0


def test_small_norms_are_not_raised():
    x = gradient(60, 60)
    x *= 1e-9 / x.norm()
    close(OR.orthogonalise(x), *model(x))


def test_same_bits_in_graphs_and_on_another_stream():
    x = gradient(6, 200, 300)
    want = OR.orthogonalise(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        assert torch.equal(OR.orthogonalise(x), want)
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = OR.orthogonalise(x)
            graphs.append((g, out))
    side.synchronize()
    x.copy_(gradient(6, 200, 300, seed=5))
    want = OR.orthogonalise(x)
    for g, _ in graphs:
        g.replay()
    with torch.cuda.stream(side):
        again = OR.orthogonalise(x)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out in graphs) and torch.equal(again, want)


# ------------------------------------------------------------------------------------------------------ optimizer step
def flat(shapes, gap=16, seed=0):
    """(groups, offsets by group, buffers) with ``gap`` elements of no matrix behind each."""
    groups, at, total = [], [], 0
    for rows, cols, n in shapes:
        here = []
        for _ in range(n):
            here.append(total)
            total += rows * cols + gap
        at.append(here)
        groups.append((rows, cols, torch.tensor(here, device=DEV)))
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda: torch.randn(total, generator=g, device=DEV)  # noqa: E731
    b = dict(master=rnd(), grad=1e-3 * rnd(), momentum=1e-3 * rnd(), ema=rnd())
    b["weights"] = b["master"].bfloat16()
    b["norm_sq"] = torch.tensor([4.0], dtype=torch.float64, device=DEV)
    return groups, at, b


ORDER = ("master", "grad", "momentum", "weights", "ema", "norm_sq")
KW = dict(lr=0.02, beta=0.9, nesterov=True, weight_decay=0.1, scale=0.2, grad_scale=0.5, max_norm=1.0, ema_beta=0.7)


def reference(groups, at, b, kw, spread):
    """({buffer: new values in 64 bits}, {buffer: what they may be off by}). ``spread``: no entry stands out of its matrix, and
    the error of an orthogonalised one is taken to be spread over its elements; else one element may have all of it (no
    element of a vector is larger than its 2-norm)."""
    clip = 1.0
    if kw["max_norm"] > 0 and b["norm_sq"] is not None:
        clip = min(1.0, kw["max_norm"] / (math.sqrt(b["norm_sq"].item()) + 1e-6))
    new = {k: b[k].double().clone() for k in ("master", "momentum", "ema")}
    off = {k: torch.zeros_like(v) for k, v in new.items()}
    for (rows, cols, _), here in zip(groups, at):
        for o in here:
            sl = slice(o, o + rows * cols)
            g = torch.nan_to_num(b["grad"][sl].double() * kw["grad_scale"] * clip, nan=0.0, posinf=1e5, neginf=-1e5)
            m0, p0, e0 = (b[k][sl].double() for k in ("momentum", "master", "ema"))
            m = kw["beta"] * m0 + (1 - kw["beta"]) * g
            u = kw["beta"] * m + (1 - kw["beta"]) * g if kw["nesterov"] else m
            x, x_off = model(u.view(rows, cols))
            rate = kw["lr"] * kw["scale"] * math.sqrt(max(rows, cols))
            p = p0 * (1 - kw["lr"] * kw["weight_decay"]) - rate * x.reshape(-1)
            new["momentum"][sl], new["master"][sl] = m, p
            off["momentum"][sl] = 8 * U32 * (m0.abs() + g.abs())
            off["master"][sl] = 8 * U32 * (p0.abs() + p.abs()) + rate * (2.0 ** -11 * x.reshape(-1).abs() + x_off.item() * (6 / math.sqrt(x.numel()) if spread else 1))
            if kw["ema_beta"] >= 0:
                new["ema"][sl] = p + kw["ema_beta"] * (e0 - p)
                off["ema"][sl] = off["master"][sl] + 8 * U32 * (e0.abs() + p.abs())
    return new, off


def check(groups, at, b, kw, zero_grad, spread=True):
    before = {k: v.clone() for k, v in b.items() if v is not None}
    new, off = reference(groups, at, b if b["ema"] is not None else {**b, "ema": torch.zeros_like(b["master"])}, kw, spread)
    OR.orthogonal_step(*(b[k] for k in ORDER), groups=groups, zero_grad=zero_grad, **kw)
    inside = torch.zeros_like(b["master"], dtype=torch.bool)
    for (rows, cols, _), here in zip(groups, at):
        for o in here:
            inside[o:o + rows * cols] = True
    for k in ("master", "momentum", "ema"):
        if b[k] is not None:
            assert bool(((b[k].double() - new[k]).abs() <= off[k] + 1e-30).all()), k
    if b["weights"] is not None:
        assert torch.equal(b["weights"][inside], b["master"][inside].bfloat16())
    assert torch.equal(b["grad"][inside], torch.zeros_like(before["grad"][inside]) if zero_grad else before["grad"][inside])
    for k, v in before.items():
        if k != "norm_sq":
            assert torch.equal(b[k][~inside], v[~inside]), k


@pytest.mark.parametrize("shapes", [[(1, 1, 1)], [(64, 64, 5)], [(48, 96, 2), (96, 48, 3)], [(33, 57, 3), (57, 33, 2), (20, 20, 4)],
                                    [(30, 500, 3), (500, 30, 2), (30, 700, 1), (40, 30, 2), (600, 30, 1)],
                                    [(130, 70, 1), (128, 300, 2)]])
@pytest.mark.parametrize("gap", [0, 1, 16])
def test_step(shapes, gap):
    groups, at, b = flat(shapes, gap)
    check(groups, at, b, KW, True)


@pytest.mark.parametrize("over", [dict(nesterov=False), dict(max_norm=0.0), dict(ema_beta=-1.0), dict(max_norm=1e9),
                                  dict(weight_decay=0.0), dict(beta=0.0)])
def test_step_settings(over):
    groups, at, b = flat([(40, 72, 3)])
    check(groups, at, b, {**KW, **over}, False)


def test_step_without_weights_average_or_norm():
    groups, at, b = flat([(40, 72, 3)])
    b["weights"] = b["ema"] = b["norm_sq"] = None
    check(groups, at, b, KW, True)


def test_step_cleans_gradients():
    groups, at, b = flat([(40, 40, 2)])
    b["grad"][5], b["grad"][77] = float("nan"), float("inf")
    b["grad"][1700] = -float("inf")
    # the infinities become 1e5 among gradients of 1e-3: each of the two matrices is next to nothing but that entry, whose
    # roundings (a relative error of the singular value 1) are all in one element
    check(groups, at, b, KW, True, spread=False)


@pytest.mark.parametrize("bad", [-16, 5 * 400, 2 ** 40, "twice", "overlapping"])
def test_offsets_outside_or_overlapping_are_reported_and_left(bad):
    groups, at, b = flat([(20, 20, 5)], gap=0)
    off = torch.tensor(at[0], device=DEV)
    off[2] = off[1] if bad == "twice" else off[1] + 100 if bad == "overlapping" else bad
    if bad in (5 * 400, 2 ** 40):
        off = off[[0, 1, 2]]
    want = {k: v.clone() for k, v in b.items()}
    good = [o for i, o in enumerate(off.tolist()) if i != 2 and 0 <= o <= 4 * 400]
    OR.orthogonal_step(*(want[k] for k in ORDER), groups=[(20, 20, torch.tensor(good, device=DEV))], **KW)
    OR.orthogonal_step(*(b[k] for k in ORDER), groups=[(20, 20, off)], **KW)
    seen = _l.status_word().item()
    _l.status_word().zero_()
    assert seen == 6
    for k in ("momentum", "grad"):
        assert torch.equal(b[k], want[k]), k
    _, _, fresh = flat([(20, 20, 5)], gap=0)
    outside = torch.ones(2000, dtype=torch.bool, device=DEV)
    for o in good:
        outside[o:o + 400] = False
    # the others of a failed call may have been updated or not
    assert torch.equal(b["master"][outside], fresh["master"][outside]) and torch.equal(b["weights"][outside], fresh["weights"][outside])


@pytest.mark.parametrize("rows,cols", [(20, 30), (150, 160), (40, 700)])          # in one launch, in many, on the Gram matrix alone
@pytest.mark.parametrize("back", [0, 1, 63, 64, "size", "behind"])
def test_offsets_whose_ends_pass_64_bits_are_reported_and_left(rows, cols, back):
    """A matrix that starts less than its size before 2^63, such as the largest integer for "no matrix": its end is no 64-bit
    number."""
    n, last = rows * cols, torch.iinfo(torch.int64).max
    bad = last - (n if back == "size" else n + 1 if back == "behind" else back)
    groups, at, b = flat([(rows, cols, 3)], gap=0)
    off = torch.tensor([0, n, bad], device=DEV)
    want = {k: v.clone() for k, v in b.items()}
    OR.orthogonal_step(*(want[k] for k in ORDER), groups=[(rows, cols, off[:2])], **KW)
    assert _l.status_word().item() == 0
    for table in ([(rows, cols, off)], [(rows, cols, off[:2]), (cols, rows, off[2:])]):      # among its kind, as a group of its own
        new = {k: v.clone() for k, v in b.items()}
        OR.orthogonal_step(*(new[k] for k in ORDER), groups=table, **KW)
        seen = _l.status_word().item()
        _l.status_word().zero_()
        assert seen == 6
        for k in ("momentum", "grad"):
            assert torch.equal(new[k], want[k]), k
        for k in ("master", "weights", "ema"):               # the others of a failed call may have been updated or not
            assert torch.equal(new[k][2 * n:], b[k][2 * n:]), k
            for i in (slice(0, n), slice(n, 2 * n)):
                assert torch.equal(new[k][i], b[k][i]) or torch.equal(new[k][i], want[k][i]), k


@pytest.mark.parametrize("rows,cols", [(20, 30), (150, 160)])          # in one launch, in many
def test_a_matrix_in_two_groups_is_reported(rows, cols):
    n = rows * cols
    for second, bad in ((n, False), (n - 1, True), (0, True)):
        b = {k: torch.zeros(3 * n + 8, device=DEV) for k in ("master", "grad", "momentum")}
        groups = [(rows, cols, torch.tensor([0, 2 * n + 4], device=DEV)), (cols, rows, torch.tensor([second], device=DEV))]
        OR.orthogonal_step(b["master"], b["grad"], b["momentum"], None, None, None, groups=groups, **KW)
        seen = _l.status_word().item()
        _l.status_word().zero_()
        assert seen == (6 if bad else 0)


def test_matrices_beyond_32_bit_offsets():
    base = torch.empty(2 ** 32 + 2 ** 20, dtype=torch.bfloat16, device=DEV)
    for rows, cols in ((64, 80), (200, 300)):
        x = base.as_strided((2, rows, cols), (2 ** 32, cols, 1))
        x.copy_(gradient(2, rows, cols))
        want = OR.orthogonalise(x.clone())
        assert torch.equal(OR.orthogonalise(x), want)
        OR.orthogonalise(x.clone(), out=x)
        assert torch.equal(x, want)


def test_two_calls_at_once():
    """On streams of their own, without waiting for one another: neither's workspace is the other's."""
    a, b = gradient(6, 200, 600), gradient(8, 300, 500, seed=3)
    want = OR.orthogonalise(a), OR.orthogonalise(b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for k, (s, x) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[k].append(OR.orthogonalise(x))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(g, want[k]) for g in got[k])


def test_batches_of_a_small_workspace_give_the_same_bits(monkeypatch):
    shapes = [(64, 64, 7), (64, 200, 3), (200, 64, 4)]
    groups, at, b = flat(shapes)
    want = {k: v.clone() for k, v in b.items()}
    OR.orthogonal_step(*(want[k] for k in ORDER), groups=groups, **KW)
    monkeypatch.setattr(OR, "WORKSPACE_BYTES", 3 * 200000)
    OR.orthogonal_step(*(b[k] for k in ORDER), groups=groups, **KW)
    for k in ORDER:
        assert torch.equal(b[k], want[k]), k
    x = gradient(7, 64, 64)
    many = OR.orthogonalise(x)
    monkeypatch.undo()
    assert torch.equal(many, OR.orthogonalise(x))


def test_step_in_a_graph():
    groups, at, b = flat([(64, 96, 4), (96, 64, 2)])
    start = {k: v.clone() for k, v in b.items()}
    eager = {k: v.clone() for k, v in b.items()}
    call = lambda bufs: OR.orthogonal_step(*(bufs[k] for k in ORDER), groups=groups, zero_grad=False, **KW)  # noqa: E731
    for _ in range(3):
        call(eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            call(b)
    side.synchronize()
    for k, v in start.items():
        b[k].copy_(v)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for k in ORDER:
        assert torch.equal(b[k], eager[k]), k
