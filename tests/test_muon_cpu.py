"""Orthogonalised updates and norms of q and k in the model, the optimizer, the configuration and checkpoints, on the CPU path."""
import math

import pytest
import torch

from aeris_gb_b200.engine import checkpoint as CK
from aeris_gb_b200.engine.init import init_params
from aeris_gb_b200.engine.optim import FlatOptimizer, OptimConfig, block_matrices, require_adamw
from aeris_gb_b200.engine.trainer import DiffusionConfig, Trainer
from aeris_gb_b200.models import oracle as O
from aeris_gb_b200.models.aeris import AerisConfig, AerisModel
from aeris_gb_b200.utils import config as C

CFG = dict(img=(16, 32), window=(8, 8), in_channels=10, out_channels=6, dim=32, heads=2, head_dim=16, mlp_dim=48, n_layers=2,
           sublayers=1, model_dtype=torch.float32, norm_eps=1e-5)


def model(seed=0, **over):
    torch.manual_seed(seed)
    return AerisModel(AerisConfig(**{**CFG, **over}))


def optim(m, **over):
    return FlatOptimizer(m, OptimConfig(**{**dict(method="muon", lr=1e-2, lr_rampup_img=0, weight_decay=0.1, decay_policy="all"), **over}))


# ------------------------------------------------------------------------------------------------------ norms of q and k
def test_modules_and_keys():
    plain, normed = model(), model(qk_norm=True)
    extra = set(normed.state_dict()) - set(plain.state_dict())
    assert extra == {f"layers.{i}.modulelist.0.1.{n}_norm.weight" for i in range(2) for n in "qk"}
    assert not set(plain.state_dict()) - set(normed.state_dict())
    assert all(torch.equal(v, normed.state_dict()[k]) for k, v in plain.state_dict().items())     # the same random draws
    assert normed.cfg.param_count() - plain.cfg.param_count() == 2 * 2 * 16


@pytest.mark.parametrize("rope", [False, True])
def test_oracle_attention_norms_before_it_rotates(rope):
    torch.manual_seed(1)
    nw, L, H, d = 2, 8, 2, 16
    qkv, wq, wk = torch.randn(nw * L, 3 * H * d), 1 + 0.2 * torch.randn(d), 1 + 0.2 * torch.randn(d)
    angles = O.rope_2d_cache(2, 4, d) if rope else None
    got = O.window_attention(qkv, nw, L, H, d, rope=angles, qk=(wq, wk, 1e-5)).double()
    q, k, v = qkv.double().view(nw, L, 3, H, d).permute(2, 0, 3, 1, 4)
    q, k = (x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double() for x, w in ((q, wq), (k, wk)))
    if rope:
        z = torch.complex(angles[0].double(), angles[1].double())
        q, k = (torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (d // 2, 2)).contiguous()) * z).flatten(-2) for x in (q, k))
    o = (q @ k.mT / math.sqrt(d)).softmax(-1) @ v
    assert (got - o.permute(0, 2, 1, 3).reshape(nw * L, H * d)).abs().max() < 1e-5


def test_init_leaves_the_norms_at_one_and_modes_without_conditioning_have_them():
    m = model(qk_norm=True)
    init_params(m, m.cfg, {"init_scale_test15": True})
    assert all(bool((p == 1).all()) for n, p in m.named_parameters() if "q_norm" in n or "k_norm" in n)
    plain = model(qk_norm=True, diffusion=False)
    y = plain(torch.randn(1, 16, 32, 10), None)
    y.square().sum().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for n, p in plain.named_parameters() if "q_norm" in n)


# ------------------------------------------------------------------------------------------------------ optimizer
def test_matrices_of_a_model():
    m = model(qk_norm=True)
    got = block_matrices(m)
    assert len(got) == 2 * 4
    assert got["layers.0.modulelist.0.1.to_qkv.weight"] == [(i * 32 * 32, 32, 32) for i in range(3)]
    assert got["layers.1.modulelist.0.3.w1.weight"] == [(0, 48, 32), (48 * 32, 48, 32)]
    assert got["layers.1.modulelist.0.3.w2.weight"] == [(0, 32, 48)]
    assert not any("latent" in k or "modulation" in k or "head" in k for k in got)


def test_step_equals_the_formula_and_leaves_the_rest_to_adamw():
    """In 64 bits, with the clipping in force. fp32 roundings of the iteration (2^-24 a step, amplified by up to 3.4445^5 = 485
    and summed over rows of 48) stay below 1e-3 of an update of lr = 1e-2."""
    m, ref = model(qk_norm=True), model(qk_norm=True)
    opt, adam = optim(m, use_ema=True), optim(ref, method="adamw", use_ema=True)
    g = torch.Generator().manual_seed(5)
    grads = {n: torch.randn(p.shape, generator=g) for n, p in m.named_parameters() if p.requires_grad}
    start = {n: p.detach().double().clone() for n, p in m.named_parameters()}
    for mod, o in ((m, opt), (ref, adam)):
        for n, p in mod.named_parameters():
            if p.requires_grad:
                p.main_grad.copy_(grads[n])
        o.step(1, 0.5, o.grad_norm_sq(0.5))
    total = math.sqrt(sum(float((0.5 * t.double()).square().sum()) for t in grads.values()))
    clip = min(1.0, opt.cfg.grad_clip_max_norm / (total + 1e-6))
    a, b, c = O.ORTHO_COEFFICIENTS
    parts, lr = block_matrices(m), opt.last_lr
    for n, p in m.named_parameters():
        if n not in parts:
            assert torch.equal(p, dict(ref.named_parameters())[n]), n
            continue
        for off, rows, cols in parts[n]:
            u = grads[n].double().reshape(-1)[off:off + rows * cols].view(rows, cols) * 0.5 * clip
            u = 0.95 * 0.05 * u + 0.05 * u
            x = u if rows <= cols else u.T
            x = x / x.norm()
            for _ in range(5):
                s = x @ x.T
                x = a * x + (b * s + c * s @ s) @ x
            x = x if rows <= cols else x.T
            want = start[n].reshape(-1)[off:off + rows * cols].view(rows, cols) * (1 - lr * 0.1) - lr * 0.2 * math.sqrt(max(rows, cols)) * x
            got = p.detach().double().reshape(-1)[off:off + rows * cols].view(rows, cols)
            assert (got - want).abs().max() < 1e-3 * lr, n
    assert all(float(x.abs().max()) == 0 for x in opt.grad_buffers())


def test_state_goes_through_a_checkpoint_and_other_methods_are_refused(tmp_path):
    m = model(qk_norm=True)
    opt = optim(m)
    for s in range(2):
        for p in m.parameters():
            if p.requires_grad:
                p.main_grad.normal_(generator=torch.Generator().manual_seed(s))
        opt.step(1, 1.0, None)
    CK.save_stage_checkpoint(str(tmp_path / "muon"), m, opt)
    m2 = model(seed=9, qk_norm=True)
    opt2 = optim(m2)
    assert CK.load_stage_checkpoint(str(tmp_path / "muon"), m2, opt2, "cpu")
    assert opt2.step_count == 2
    for (k, v), (k2, v2) in zip(sorted(opt.state_dict()["exp_avg"].items()), sorted(opt2.state_dict()["exp_avg"].items())):
        assert k == k2 and torch.equal(v, v2)
    assert all(torch.equal(a, b) for a, b in zip(m.parameters(), m2.parameters()))
    m3 = model(qk_norm=True)
    adam = optim(m3, method="adamw")
    before = [p.detach().clone() for p in m3.parameters()]
    with pytest.raises(ValueError, match="another method"):
        CK.load_stage_checkpoint(str(tmp_path / "muon"), m3, adam, "cpu")
    assert all(torch.equal(a, b) for a, b in zip(before, m3.parameters())) and adam.step_count == 0
    CK.save_stage_checkpoint(str(tmp_path / "adamw"), m3, adam)
    with pytest.raises(ValueError, match="another method"):
        CK.load_stage_checkpoint(str(tmp_path / "adamw"), m2, opt2, "cpu")
    with pytest.raises(ValueError, match="another method"):
        opt2.load_state_dict(adam.state_dict())


@pytest.mark.parametrize("method", ["adamw", "muon"])
def test_states_in_part_are_loaded_in_part(method):
    """Moments that are not there are left as they are; a momentum without second moments is refused by AdamW alone."""
    m, other = model(), model(seed=3)
    opt, src = optim(m, method=method), optim(other, method=method)
    for s in src.segments:
        s.m.normal_()
        if s.v is not None:
            s.v.uniform_()
    src.step_count, src.cur_nimg = 3, 7
    sd = src.state_dict()
    clone = lambda: {k: {n: t.clone() for n, t in opt._named_views(k).items()} for k in "mv"}  # noqa: E731
    for first, second in ((None, None), (None, sd["exp_avg_sq"]), (sd["exp_avg"], None), (sd["exp_avg"], {}),
                          ({}, sd["exp_avg_sq"]), (dict(list(sd["exp_avg"].items())[:2]), sd["exp_avg_sq"])):
        before = clone()
        opt.load_state_dict({**sd, "exp_avg": first, "exp_avg_sq": second})
        after = clone()
        for k, given in (("m", first), ("v", second)):
            for n, t in after[k].items():
                assert torch.equal(t, (given if given and n in given else before[k])[n]), (k, n)
        assert (opt.step_count, opt.cur_nimg) == (3, 7)
        for s in opt.segments:
            s.m.zero_()


def test_a_momentum_alone_is_refused_by_adamw_and_untouched():
    muon, adam = optim(model()), optim(model(), method="adamw")
    muon.step_count = 5
    for s in muon.segments:
        s.m.normal_()
    with pytest.raises(ValueError, match="another method"):
        adam.load_state_dict(muon.state_dict())
    assert adam.step_count == 0 and all(float(s.m.abs().max()) == 0 for s in adam.segments)


def test_a_file_without_any_second_moments_is_not_loaded(tmp_path):
    m = model()
    opt = optim(m, method="adamw")
    path, = CK.save_stage_checkpoint(str(tmp_path), m, opt)[:1]
    file = torch.load(path, weights_only=True)
    for st in file["optimizer_state_dict"]["state"].values():
        del st["exp_avg_sq"]
    file.pop("integrity")
    torch.save(file, path)
    assert CK.load_stage_checkpoint(str(tmp_path), m, opt, "cpu") is False


def test_unknown_method_and_optimizers_that_cut_matrices():
    with pytest.raises(ValueError, match="method"):
        optim(model(), method="sgd")
    with pytest.raises(ValueError, match="whole matrices"):
        require_adamw(OptimConfig(method="muon"), "it")
    from aeris_gb_b200.engine.dist_optim import DistOptimizer
    with pytest.raises(ValueError, match="whole matrices"):
        DistOptimizer(model(), OptimConfig(method="muon"), None)


def test_training_steps():
    cfg = AerisConfig(**CFG, qk_norm=True)
    tr = Trainer(cfg, OptimConfig(method="muon", lr=1e-3, lr_rampup_img=0), DiffusionConfig(cond_channels=4), "cpu")
    before = {n: p.detach().clone() for n, p in tr.model.named_parameters()}
    for i in range(2):
        loss = tr.train_step(torch.randn(1, 16, 32, 6), torch.randn(1, 16, 32, 4))
        assert math.isfinite(loss)
    for n in block_matrices(tr.model):
        assert not torch.equal(before[n], dict(tr.model.named_parameters())[n])
        assert bool(dict(tr.model.named_parameters())[n].isfinite().all())


# ------------------------------------------------------------------------------------------------------ configuration
def test_configuration():
    cfg = C.compose("train", ["experiment=tiny_cpu", "optimizer._target_=torch.optim.Muon", "model.qk_norm=true",
                              "optimizer.momentum=0.9", "optimizer.ns_steps=4"])
    o = C.optim_config(cfg)
    assert (o.method, o.muon_beta, o.muon_nesterov, o.muon_steps, o.muon_scale) == ("muon", 0.9, True, 4, 0.2)
    assert C.model_config(cfg).qk_norm
    plain = C.compose("train", ["experiment=tiny_cpu"])
    assert C.optim_config(plain).method == "adamw" and not C.model_config(plain).qk_norm
    group = C.compose("train", ["optimizer=muon", "experiment=b200_wp_inference"])
    assert C.optim_config(group).method in ("muon", "adamw")       # an experiment's own optimizer section comes later


def experiments():
    return sorted(p.stem for p in (C.CONFIG_ROOT / "experiment").glob("*.yaml"))


@pytest.mark.parametrize("experiment", experiments())
def test_the_group_selects_the_method_with_every_experiment(experiment):
    """Whose other optimizer keys stand."""
    plain = C.optim_config(C.compose("train", [f"experiment={experiment}"]))
    group = C.optim_config(C.compose("train", ["optimizer=muon", f"experiment={experiment}"]))
    assert plain.method == "adamw" and group.method == "muon"
    assert (group.lr, group.betas, group.weight_decay, group.eps) == (plain.lr, plain.betas, plain.weight_decay, plain.eps)
    assert (group.muon_beta, group.muon_nesterov, group.muon_steps, group.muon_scale) == (0.95, True, 5, 0.2)
    back = C.compose("train", ["optimizer=muon", f"experiment={experiment}", "optimizer._target_=torch.optim.AdamW"])
    assert C.optim_config(back).method == "adamw"                  # a key on the command line comes last
    assert C.optim_config(C.compose("train", ["optimizer=muon"])).method == "muon"
    assert C.optim_config(C.compose("train", ["optimizer=adamw", f"experiment={experiment}"])) == plain


def test_a_selected_target_stands_against_an_experiment_of_another(tmp_path):
    for group in ("optimizer", "experiment"):
        (tmp_path / group).mkdir()
    (tmp_path / "train.yaml").write_text("defaults:\n  - _self_\n  - optimizer: a\n  - experiment: x\n")
    (tmp_path / "optimizer" / "a.yaml").write_text("_target_: A\nlr: 1.0\nown: 2\n")
    (tmp_path / "optimizer" / "b.yaml").write_text("lr: 3.0\n")
    (tmp_path / "experiment" / "x.yaml").write_text("# @package _global_\noptimizer:\n  _target_: X\n  lr: 5.0\n")
    section = lambda *o: C.compose("train", list(o), tmp_path).optimizer.to_dict()  # noqa: E731
    assert section() == {"_target_": "X", "lr": 5.0, "own": 2}
    assert section("optimizer=a") == {"_target_": "A", "lr": 5.0, "own": 2}
    assert section("optimizer=b") == {"_target_": "X", "lr": 5.0}
    assert section("optimizer=a", "optimizer._target_=Y")["_target_"] == "Y"


@pytest.mark.parametrize("key", ["ns_coefficients=[3.4445,-4.775,2.0315]", "adjust_lr_fn=match_rms_adamw", "adjust_lr_fn=original",
                                 "momentun=0.9"])
def test_keys_that_the_orthogonalised_updates_do_not_take_are_refused(key):
    name = key.partition("=")[0]
    cfg = C.compose("train", ["experiment=tiny_cpu", "optimizer=muon", f"+optimizer.{key}"])
    with pytest.raises(ValueError, match=f"optimizer.{name}"):
        C.optim_config(cfg)
    C.optim_config(C.compose("train", ["experiment=tiny_cpu", f"+optimizer.{key}"]))       # AdamW's sections as before
