"""Refusals of the orthogonalisation and of the optimizer step on it: made on the host, before anything is launched."""
import pytest
import torch

from aeris_gb_b200.ops import orthogonalise as OR


@pytest.mark.parametrize("x,kw", [
    (torch.randn(4), {}), (torch.randn(2, 2, 4, 4), {}), (torch.randn(4, 4).half(), {}), (torch.randn(4, 4).double(), {}),
    (torch.randn(4, 4), dict(steps=0)), (torch.randn(4, 4), dict(steps=21)), (torch.randn(4, 4), dict(steps=2.0)),
    (torch.randn(4, 4), dict(out=torch.empty(4, 4))), (torch.randn(4, 4), dict(out=torch.empty(4, 5).bfloat16())),
    (torch.randn(4, 4), dict(out=torch.empty(1, 4).bfloat16().expand(4, 4))),
    (torch.randn(2, 4, 4), dict(out=torch.empty(1, 4, 4).bfloat16().expand(2, 4, 4))),
    (torch.randn(4, 4), dict(out=torch.empty(4, 4).bfloat16().t())),
    (torch.randn(4, 4), dict(eps=0.0)), (torch.randn(4, 4), dict(eps=-1e-7)), (torch.randn(4, 4), dict(eps=float("nan"))),
    (torch.randn(1).expand(1, 2 ** 30 + 1), {}), (torch.randn(1).expand(2 ** 30 + 1, 1), {}),
    (torch.randn(4, 4), {}),                                                     # not on a GPU
])
def test_orthogonalise_refuses(x, kw):
    with pytest.raises(ValueError):
        OR.orthogonalise(x, **kw)


N = 64


def step(**over):
    a = dict(master=torch.zeros(N), grad=torch.zeros(N), momentum=torch.zeros(N), weights=torch.zeros(N).bfloat16(),
             ema=torch.zeros(N), norm_sq=torch.zeros(1, dtype=torch.float64), groups=[(4, 4, torch.tensor([0, 16]))])
    kw = dict(lr=1e-3, beta=0.9, nesterov=True, weight_decay=0.1, scale=0.2, grad_scale=1.0, max_norm=1.0, ema_beta=0.5)
    for k, v in over.items():
        (a if k in a else kw)[k] = v
    groups = a.pop("groups")
    OR.orthogonal_step(*a.values(), groups=groups, **kw)


@pytest.mark.parametrize("bad", [
    dict(master=torch.zeros(8, 8)), dict(master=torch.zeros(N).bfloat16()), dict(master=torch.zeros(2 * N)[::2]),
    dict(master=torch.zeros(N + 1)[1:]), dict(grad=torch.zeros(N + 1)), dict(grad=torch.zeros(N).bfloat16()),
    dict(momentum=torch.zeros(2 * N)[::2]), dict(momentum=torch.zeros(N + 1)[1:]), dict(weights=torch.zeros(N)),
    dict(ema=torch.zeros(N - 1)), dict(norm_sq=torch.zeros(1)), dict(norm_sq=torch.zeros(2, dtype=torch.float64)),
    dict(groups=[(0, 4, torch.tensor([0]))]), dict(groups=[(4, 4, torch.tensor([0], dtype=torch.int32))]),
    dict(groups=[(4, 4, torch.tensor([[0]]))]), dict(groups=[(4, 4, torch.tensor([0, 1, 2, 3])[::2])]),
    dict(groups=[(4, 4, torch.tensor([0, 16, 32, 48, 64]))]), dict(groups=[(9, 9, torch.tensor([0]))]), dict(steps=0),
    dict(eps=0.0), dict(groups=[(1, 2 ** 30 + 1, torch.tensor([], dtype=torch.int64))]),
    {},                                                                           # not on a GPU
])
def test_step_refuses(bad):
    with pytest.raises(ValueError):
        step(**bad)


@pytest.mark.parametrize("strides,shape,fine", [((32, 8, 1), (2, 4, 8), True), ((32, 7, 1), (2, 4, 8), False),
                                                ((32, 0, 1), (2, 4, 8), False), ((32, 1, 4), (2, 4, 8), False),
                                                ((0, 2 ** 31 - 1, 1), (2, 4, 8), True), ((0, 2 ** 31, 1), (2, 4, 8), False),
                                                ((0, 2 ** 40, 1), (2, 1, 8), True), ((0, 9, 5), (2, 4, 1), True)])
def test_pitches_that_the_kernels_count(strides, shape, fine):
    assert OR._pitched(torch.empty(1, device="meta").as_strided(shape, strides)) == fine


def test_results_over_the_input_are_refused():
    x = torch.randn(3, 4, 8).bfloat16()
    wide = torch.zeros(3, 4, 16).bfloat16()
    for inp, out, fine in ((x, x, False), (x, x.clone(), True), (x, x[:1].clone().expand(3, 4, 8), False),
                           (wide[:, :, :8], wide[:, :, 8:], True), (wide[:, :, :8], wide[:, :, 4:12], False),
                           (wide[:2, :, :8], wide[1:, :, :8], False), (wide[:1, :, :8], wide[1:2, :, :8], True),
                           (torch.randn(4, 8), torch.empty(4, 8).bfloat16(), True)):
        with pytest.raises(ValueError) as e:
            OR.orthogonalise(inp, out=out)
        assert ("on a GPU" in str(e.value)) == fine, e.value


@pytest.mark.parametrize("a,b", [("master", "grad"), ("grad", "momentum"), ("master", "ema"), ("ema", "momentum")])
@pytest.mark.parametrize("by", [0, 4, N - 4])
def test_buffers_of_a_step_that_share_memory_are_refused(a, b, by):
    whole = torch.zeros(2 * N)
    with pytest.raises(ValueError, match="share memory"):
        step(**{a: whole[:N], b: whole[by:by + N]})
    with pytest.raises(ValueError, match="share memory"):
        step(**{a: whole[:N], "weights": whole[by:by + N].view(torch.bfloat16)[:N]})
    with pytest.raises(ValueError, match="on a GPU"):
        step(**{a: whole[:N], b: whole[N:]})
