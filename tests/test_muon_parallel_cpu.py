"""Orthogonalised updates and norms of q and k in the pipeline engine, over gloo ranks, against one process.

Tolerance: gradients of another split differ by the order of fp32 sums, about 1e-6 of their norm. Five steps raise what lies in small
singular directions by up to 3.4445^5 = 485, and an update is 0.01 * 0.2 * sqrt(64) = 0.016 times the result: 8e-6 a step, two steps,
and as much again for the weights that the second gradient is taken at."""
import dataclasses
import tempfile

import pytest
import test_engine_gloo as base

PLAIN_RUN, PLAIN_CFG, PLAIN_OPTIM = base._run, base._cfg, base.OptimConfig


def _cfg(*args):
    return dataclasses.replace(PLAIN_CFG(*args), qk_norm=True)


def _optim(**kw):
    return PLAIN_OPTIM(**{**kw, "lr": 0.01, "method": "muon"})


def _run(rank, *args):
    base._cfg, base.OptimConfig = _cfg, _optim
    try:
        PLAIN_RUN(rank, *args)
    finally:
        base._cfg, base.OptimConfig = PLAIN_CFG, PLAIN_OPTIM


@pytest.fixture
def launch(monkeypatch):
    monkeypatch.setattr(base, "_run", _run)
    return base._launch


@pytest.fixture(scope="module")
def single():
    kept = base._run
    base._run = _run
    try:
        return base._launch(1, PP=1, WP=(1, 1), gas=4, iters=2)
    finally:
        base._run = kept


@pytest.mark.parametrize("world,kw", [(2, dict(PP=1, WP=(1, 1), gas=2)), (4, dict(PP=2, WP=(1, 2), gas=4, overlap=True)),
                                      (2, dict(PP=1, WP=(1, 1), SP=2, gas=4))], ids=["data", "pipeline and windows", "sequence"])
def test_splits_match_one_process(single, launch, world, kw):
    sd, _, norm = launch(world, iters=2, **kw)
    assert any("q_norm" in k for stage in sd.values() for k in stage)
    base._assert_same(sd, single[0], tol=5e-5)
    assert norm == pytest.approx(single[2], rel=1e-4)


def test_checkpoint_resumes_on_another_split(single, launch):
    where = tempfile.mkdtemp()
    launch(1, PP=1, WP=(1, 1), gas=4, iters=1, ckpt_dir=where)
    sd, _, _ = launch(2, PP=2, WP=(1, 1), gas=4, iters=1, ckpt_dir=where, resume=True)
    base._assert_same(sd, single[0], tol=5e-5)


def test_sharded_optimizer_is_refused(launch):
    with pytest.raises(ValueError, match="whole matrices"):
        launch(1, PP=1, WP=(1, 1), gas=4, iters=1, distopt=True)
