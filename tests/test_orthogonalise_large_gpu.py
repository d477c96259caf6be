"""Orthogonalisation where products go by CTA pairs, where two steps share an update, and where a batch has two lengths, against the
formula in 64 bits.

Tolerance as in ``test_orthogonalise_gpu.py``: twice the largest distance of eight runs of the formula in which every stored array
is off by up to half a step of fp16. Where two steps share an update other arrays are stored, with S the Gram matrix and P = a I +
b S + c S^2: T = P S, S' = T P, P' = a I + b S' + c S'^2, Q = P' P, and X <- Q X. Square factors are stored symmetric.
"""
import pytest
import torch

import test_orthogonalise_gpu as small
from aeris_gb_b200.ops import lib as _l
from aeris_gb_b200.ops import orthogonalise as OR
from test_orthogonalise_gpu import DEV, KW, ORDER, A, B, C, close, flat, gradient, noisy

pytestmark = pytest.mark.gpu


def groups_of(steps, two):
    sizes, left = [], steps
    while left:
        sizes.append(2 if two and left > 1 and len(sizes) % 2 == 0 else 1)
        left -= sizes[-1]
    return sizes


def iterate(x, sizes, eps, g=None):
    if x.shape[-2] > x.shape[-1]:
        return iterate(x.mT, sizes, eps, g).mT
    def sym(t):  # noqa: E306
        t = noisy(t, g, 512).tril()
        return t + t.tril(-1).mT
    one = torch.eye(x.shape[-2], dtype=torch.float64, device=DEV)
    x = noisy(x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(eps), g, 512)
    for n in sizes:
        s = sym(x @ x.mT)
        p = sym(A * one + B * s + C * (s @ s))
        if n == 2:
            s = sym(sym(p @ s) @ p)
            p = sym(sym(A * one + B * s + C * (s @ s)) @ p)
        x = noisy(p @ x, g, 512)
    return x


def model(x, sizes, eps=1e-7):
    """(exact result, 2-norm that each matrix may be off by before its last rounding)."""
    x = x.double()
    want = iterate(x, sizes, eps)
    off = torch.zeros((*x.shape[:-2], 1, 1), dtype=torch.float64, device=DEV)
    for k in range(8):
        d = iterate(x, sizes, eps, torch.Generator(device=DEV).manual_seed(k)) - want
        off = torch.maximum(off, d.square().sum((-2, -1), keepdim=True).sqrt())
    return want, 2 * off


GRAM, FACTOR, UPDATE, TWO, PARTS = "gram pairs", "factor pairs", "update pairs", "two steps", "gram parts"
# sides that are no multiples of 256, so that both CTAs of a pair have tiles that end early
BATCHES = [((16, 1500, 1500), {GRAM, FACTOR, UPDATE}), ((6, 1030, 4100), {TWO, UPDATE}), ((8, 650, 1300), {TWO, GRAM, UPDATE}),
           ((8, 1300, 650), {TWO, GRAM, UPDATE}), ((20, 400, 1030), {TWO, GRAM}), ((100, 385, 385), {UPDATE}),
           ((1, 1900, 1800), {TWO, UPDATE}), ((42, 384, 1024), {TWO}), ((2, 385, 387), {TWO}), ((7, 151, 4472), {PARTS, UPDATE}),
           ((1, 390, 9000), {TWO, PARTS})]


def shapes_alone(v):
    return "-".join(sorted(v)) if isinstance(v, set) else str(v)


@pytest.mark.parametrize("shape,route", BATCHES, ids=shapes_alone)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_batches(shape, route, dt):
    count, rows, cols = shape
    assert OR.route([(rows, cols, count)]) == route
    x = gradient(*shape).to(dt)
    got = OR.orthogonalise(x)
    close(got, *model(x, groups_of(5, TWO in route)))
    assert torch.equal(OR.orthogonalise(x), got)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 8])
@pytest.mark.parametrize("shape,route", [((400, 700), {TWO}), ((700, 400), {TWO}), ((20, 400, 1030), {TWO, GRAM})], ids=shapes_alone)
def test_steps(steps, shape, route):
    """Odd and even numbers of groups: the result lies in either of the two X."""
    count = shape[0] if len(shape) == 3 else 1
    assert OR.route([(*shape[-2:], count)], steps) == (route if steps > 1 else route - {TWO})
    x = gradient(*shape)
    close(OR.orthogonalise(x, steps=steps), *model(x, groups_of(steps, True), 1e-7))


@pytest.mark.parametrize("shape", [(400, 700), (390, 2000), (1500, 390), (8, 650, 1300)])
@pytest.mark.parametrize("noise", [0.0, 0.1, 10.0])
def test_spectra(shape, noise):
    x = gradient(*shape, noise=noise)
    close(OR.orthogonalise(x), *model(x, groups_of(5, True)))


@pytest.mark.parametrize("rank", [1, 4, 60])
@pytest.mark.parametrize("rows,cols", [(400, 900), (390, 390), (1200, 500)])
def test_low_rank(rank, rows, cols):
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(rows, rank, generator=g, device=DEV) @ torch.randn(rank, cols, generator=g, device=DEV)
    close(OR.orthogonalise(x), *model(x, groups_of(5, rows != cols)))


@pytest.mark.parametrize("shapes,route", [
    ([(400, 400, 3), (400, 900, 2), (900, 400, 2)], {TWO}),
    ([(130, 130, 3), (130, 500, 2), (500, 130, 1)], set()),
    ([(1030, 1030, 8), (1030, 2100, 3), (2100, 1030, 3)], {TWO, GRAM, FACTOR, UPDATE}),
    ([(1100, 2500, 2), (1100, 1100, 2)], {TWO, GRAM, FACTOR}),
    ([(900, 900, 20), (910, 900, 2)], {TWO, GRAM, FACTOR, UPDATE}),
    ([(300, 900, 2), (700, 300, 2), (300, 400, 1), (300, 300, 2)], None)], ids=shapes_alone)          # more lengths than a batch takes
@pytest.mark.parametrize("gap", [1, 16])
def test_step_with_two_lengths(shapes, route, gap, monkeypatch):
    if route is not None:
        assert OR.route(shapes) == route
    groups, at, b = flat(shapes, gap)
    monkeypatch.setattr(small, "model", lambda x: model(x, groups_of(5, TWO in (route or ()))))
    small.check(groups, at, b, KW, True)


def test_step_by_pairs_in_a_graph_and_on_another_stream():
    shapes = [(1030, 1030, 8), (1030, 2100, 6)]
    groups, _, b = flat(shapes)
    start = {k: v.clone() for k, v in b.items()}
    call = lambda bufs: OR.orthogonal_step(*(bufs[k] for k in ORDER), groups=groups, zero_grad=False, **KW)  # noqa: E731
    eager = {k: v.clone() for k, v in b.items()}
    for _ in range(2):
        call(eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            call(b)
        for k, v in start.items():
            b[k].copy_(v)
        g.replay()
        call(b)
    side.synchronize()
    for k in ORDER:
        assert torch.equal(b[k], eager[k]), k
    assert _l.status_word().item() == 0
