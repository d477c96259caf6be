"""Norms of q and k inside the fused block, orthogonalised updates inside the optimizer, and both together in training steps.

Tolerance of the block: kernels and the oracle in bf16 round the same intermediate results to bf16, in places of their own; so
what the bf16 oracle is off the fp32 oracle by is what bf16 costs, and the kernels may be off by twice that."""
import math

import pytest
import torch

from aeris_gb_b200.engine.optim import FlatOptimizer, OptimConfig, block_matrices
from aeris_gb_b200.engine.trainer import DiffusionConfig, Trainer
from aeris_gb_b200.models import fused
from aeris_gb_b200.models import oracle as O
from aeris_gb_b200.models.aeris import AerisConfig, AerisModel
from aeris_gb_b200.ops import elementwise as E
from aeris_gb_b200.ops import lib as _l
from conftest import rel_err

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("n1", "to_qkv", "wo", "n2", "w1", "w2", "qn", "kn")


def operands(D, heads, d, F, B, wins, L, seed=0):
    torch.manual_seed(seed)
    rnd = lambda *s: (torch.randn(s, device=DEV) * s[-1] ** -0.5).bfloat16()  # noqa: E731
    norm = lambda n: (1 + 0.2 * torch.randn(n, device=DEV)).bfloat16()  # noqa: E731
    ws = dict(n1=norm(D), to_qkv=rnd(3 * heads * d, D), wo=rnd(D, heads * d), n2=norm(D), w1=rnd(2 * F, D), w2=rnd(D, F),
              qn=3 * norm(d), kn=norm(d))
    return torch.randn(B * wins * L, D, device=DEV).bfloat16(), 0.3 * torch.randn(B, 6 * D, device=DEV), ws


def oracle(x, mod, ws, dy, meta, dt):
    leaves = [t.to(dt).detach().requires_grad_(True) for t in (x, mod, *ws.values())]
    p = dict(zip(NAMES, leaves[2:]))
    att = lambda q, nw, nl, H, d: O.window_attention(q, nw, nl, H, d, rope=meta.rope, qk=(p["qn"], p["kn"], meta.eps))  # noqa: E731
    y = O.block_forward(leaves[0], leaves[1], p, n_win_per_sample=meta.n_win_per_sample, L=meta.L, heads=meta.heads,
                        head_dim=meta.head_dim, after_mod_norm=meta.mode == E.MODE_MOD_THEN_NORM, eps=meta.eps, attention=att)
    y.backward(dy.to(dt))
    return [y.detach(), *(t.grad for t in leaves)]


@pytest.mark.parametrize("D,heads,d,F,B,wins,win,rope,keep", [
    (128, 2, 64, 128, 2, 3, (8, 8), False, False), (256, 2, 128, 256, 1, 4, (6, 10), True, True),
    (256, 8, 32, 384, 2, 2, (15, 15), True, False), (128, 16, 8, 256, 1, 2, (4, 4), False, True)])
def test_block(D, heads, d, F, B, wins, win, rope, keep):
    L = win[0] * win[1]
    x, mod, ws = operands(D, heads, d, F, B, wins, L)
    dy = torch.randn_like(x)
    meta = fused.BlockMeta(wins, L, heads, d, E.MODE_MOD_THEN_NORM, 1e-3, 2, rope=O.rope_2d_cache(*win, d, device=DEV) if rope else None,
                           keep=keep, min_chunk_bytes=0, qk_norm=True)
    leaves = [t.clone().requires_grad_(True) for t in (x, mod, *ws.values())]
    y = fused.run_block(*leaves[:2], meta, *leaves[2:8], None, None, *leaves[8:])
    y.backward(dy.clone())
    got = [y.detach(), *(t.grad for t in leaves)]
    exact = oracle(x, mod, ws, dy, meta, torch.float32)
    low = oracle(x, mod, ws, dy, meta, torch.bfloat16)
    for name, a, b, c in zip(("y", "x", "mod", *NAMES), got, exact, low):
        assert rel_err(a, b) <= 2 * rel_err(c, b) + 2.0 ** -8, (name, rel_err(a, b), rel_err(c, b))
    with torch.no_grad():                        # without a graph: the same kernels
        assert torch.equal(fused.run_block(x, mod, meta, *list(ws.values())[:6], None, None, ws["qn"], ws["kn"]), y)


def test_block_takes_weights_with_the_option_only():
    x, mod, ws = operands(128, 2, 64, 128, 1, 1, 64)
    w = list(ws.values())
    for on, qk in ((True, ()), (False, w[6:])):
        meta = fused.BlockMeta(1, 64, 2, 64, E.MODE_MOD_THEN_NORM, 1e-3, qk_norm=on)
        with pytest.raises(ValueError, match="qk_norm"):
            fused.run_block(x, mod, meta, *w[:6], None, None, *qk)


CFG = dict(img=(30, 60), window=(15, 15), in_channels=20, out_channels=8, dim=256, heads=4, head_dim=64, mlp_dim=512, n_layers=2,
           sublayers=1, chunk_windows=3, use_rope=True, qk_norm=True)


def test_model_gradients_do_not_depend_on_what_is_kept(monkeypatch):
    torch.manual_seed(3)
    model = AerisModel(AerisConfig(**CFG)).cuda()
    for n, p in model.named_parameters():
        torch.nn.init.normal_(p, 1.0 if "_norm" in n else 0.0, std=0.05)
    x, t = torch.randn(2, 30, 60, 20, device=DEV), torch.tensor([0.4, 1.1], device=DEV)
    runs = []
    for kept in (0, 2):
        monkeypatch.setattr(fused, "plan_kept_blocks", lambda *a, kept=kept: kept)
        model.zero_grad(set_to_none=True)
        y = model(x, t)
        (y * torch.linspace(-1, 1, y.numel(), device=DEV).view_as(y)).sum().backward()
        runs.append((y.detach(), {n: p.grad.float().clone() for n, p in model.named_parameters() if p.grad is not None}))
    assert torch.equal(runs[0][0], runs[1][0])
    assert {n for n in runs[0][1] if "q_norm" in n or "k_norm" in n}
    for n, g in runs[0][1].items():
        assert rel_err(runs[1][1][n], g) < 2.0 ** -9, n      # sums in another order, rounded to bf16 once


def test_optimizer_equals_its_cpu_path():
    """Momentum to a few fp32 roundings; updates to what fp16 factors leave of an orthogonalised matrix (below 5e-3 for these
    well-conditioned gradients: their exact tolerance is tested with the operator), masters accordingly."""
    def make(dev):
        torch.manual_seed(1)
        m = AerisModel(AerisConfig(**{**CFG, "model_dtype": torch.bfloat16})).to(dev)
        return m, FlatOptimizer(m, OptimConfig(method="muon", lr=1e-2, lr_rampup_img=0, weight_decay=0.1, decay_policy="all"))
    (mg, og), (mc, oc) = make(DEV), make("cpu")
    start = {n: v.clone() for n, v in oc.master_state_dict().items()}
    gen = torch.Generator().manual_seed(2)
    for p, q in zip(mg.parameters(), mc.parameters()):
        if p.requires_grad:
            g = 1e-2 * torch.randn(p.shape, generator=gen)
            q.main_grad.copy_(g)
            p.main_grad.copy_(g)
    for o in (og, oc):
        o.step(2, 0.5, o.grad_norm_sq(0.5))
    masters, moments, cpu = og.master_state_dict(), og.state_dict()["exp_avg"], oc.state_dict()["exp_avg"]
    parts = block_matrices(mc)
    for n, want in oc.master_state_dict().items():
        got = masters[n].cpu()
        assert rel_err(moments[n].cpu(), cpu[n]) < 1e-6, n
        moved = (want - start[n]).norm()
        assert (got - want).norm() <= (5e-3 if n in parts else 1e-4) * moved + 1e-6 * want.norm(), n
    for s in og.segments:
        if s.model_flat is not None:
            assert torch.equal(s.model_flat, s.master.to(s.model_flat.dtype))
        assert float(s.grad.abs().max()) == 0


@pytest.mark.parametrize("method", ["muon", "adamw"])
def test_training_steps_run_together(method):
    """Norms, rotation, attention, orthogonalised updates and AdamW for the rest in whole steps; the second one reads what the
    first has written. Two trainers from one seed agree."""
    losses = []
    for _ in range(2):
        tr = Trainer(AerisConfig(**{**CFG, "in_channels": 20}), OptimConfig(method=method, lr=1e-3, lr_rampup_img=0),
                     DiffusionConfig(cond_channels=12), DEV)
        for n, p in tr.model.named_parameters():
            if "_norm" in n:
                assert bool((p == 1).all())
        g = torch.Generator().manual_seed(4)
        before = {n: v.clone() for n, v in tr.opt.master_state_dict().items()}
        count = _l.launch_count()
        losses.append([tr.train_step(torch.randn(2, 30, 60, 8, generator=g), torch.randn(2, 30, 60, 12, generator=g))
                       for _ in range(3)])
        assert _l.launch_count() > count
        after = tr.opt.master_state_dict()
        for n in block_matrices(tr.model):
            assert bool(after[n].isfinite().all()) and not torch.equal(after[n], before[n]), n
    assert all(math.isfinite(v) for v in losses[0])
    # gradients of both runs differ by the order of fp32 sums; a bf16 weight may land on its neighbour
    assert losses[0][0] == pytest.approx(losses[1][0], rel=1e-5) and losses[0] == pytest.approx(losses[1], rel=1e-2)


def test_sampling_applies_the_norms(monkeypatch):
    """A sampler run, which the native call does not take: one evaluation at a time, and the weights of the norms count."""
    from aeris_gb_b200.diffusion.rollout import DeviceForecaster, SamplerConfig
    from aeris_gb_b200.models.aeris import StreamContext
    from aeris_gb_b200.models.sampling import Evaluations
    torch.manual_seed(0)
    cfg = AerisConfig(**{**CFG, "in_channels": 2 * 8 + 2})
    model = AerisModel(cfg).cuda().eval()
    torch.nn.init.normal_(model.output_stage.head.weight, std=0.05)
    prepare, taken = Evaluations.prepare, []
    monkeypatch.setattr(Evaluations, "prepare", lambda *a: taken.append(prepare(*a)) or taken[-1])
    gen = torch.Generator(device=DEV).manual_seed(1)
    state, forcing = (torch.randn(2, 30, 60, c, device=DEV, generator=gen) for c in (8, 2))
    stats = {k: torch.full((8,), float("std" in k), device=DEV) for k in ("x_mean", "x_std", "t_mean", "t_std")}
    run = lambda: DeviceForecaster(model, StreamContext(cfg, 2), stats, SamplerConfig(n_steps=2), 8, seed=3).step(state, forcing)  # noqa: E731
    first = run()
    assert torch.equal(run(), first) and bool(first.isfinite().all()) and taken == [None, None]
    with torch.no_grad():
        for n, p in model.named_parameters():
            if "q_norm" in n:
                p.mul_(4)
    assert not torch.equal(run(), first)
