"""Refusals of window attention with a position bias: made on the host, before anything is launched."""
import pytest
import torch

from aeris_gb_b200.ops import position_bias as PB

W, HIGH, WIDE, H, D = 3, 2, 4, 2, 16
T, BF = W * HIGH * WIDE, torch.bfloat16
OFF = 3 * 7


def rows(cols, dt=BF, n=T):
    return torch.randn(n, cols).to(dt)


def forward(**over):
    a = dict(qkv=rows(3 * H * D), n_win=W, window=(HIGH, WIDE), heads=H, d=D, table=torch.zeros(OFF, H), buckets=None, out=None, lse=None,
             scale=None)
    a.update(over)
    return PB.biased_attn_fwd(*[a.pop(k) for k in ("qkv", "n_win", "window", "heads", "d", "table", "buckets")], **a)


def backward(**over):
    a = dict(d_o=rows(H * D), qkv=rows(3 * H * D), o=rows(H * D), lse=torch.zeros(W, H, HIGH * WIDE), n_win=W, window=(HIGH, WIDE), heads=H,
             d=D, table=torch.zeros(OFF, H), buckets=None)
    a.update(over)
    return PB.biased_attn_bwd(*[a.pop(k) for k in ("d_o", "qkv", "o", "lse", "n_win", "window", "heads", "d", "table", "buckets")], **a)


BAD = {
    "fp32": dict(qkv=rows(3 * H * D, torch.float32)),
    "other rows": dict(qkv=rows(3 * H * D, n=T + 1)),
    "columns apart": dict(qkv=torch.randn(3 * H * D, T).to(BF).t()),
    "rows that share": dict(qkv=rows(3 * H * D, n=1).expand(T, 3 * H * D)),
    "window without rows": dict(window=(0, WIDE)),
    "window of one number": dict(window=(HIGH * WIDE,)),
    "window too large": dict(window=(256, 256), n_win=0, qkv=rows(3 * H * D, n=0)),
    "wide heads": dict(d=129, qkv=rows(3 * H * 129)),
    "no heads": dict(heads=0, qkv=rows(0)),
    "too many windows": dict(n_win=65536),
    "table of other positions": dict(table=torch.zeros(OFF - 1, H)),
    "table of other heads": dict(table=torch.zeros(OFF, H + 1)),
    "table in half": dict(table=torch.zeros(OFF, H).half()),
    "table transposed": dict(table=torch.zeros(H, OFF).t()),
    "empty table": dict(table=torch.zeros(0, H), buckets=torch.zeros(OFF, dtype=torch.int32)),
    "buckets of other positions": dict(buckets=torch.zeros(OFF + 1, dtype=torch.int32)),
    "buckets in floating point": dict(buckets=torch.zeros(OFF)),
    "buckets with gaps": dict(buckets=torch.zeros(2 * OFF, dtype=torch.int64)[::2]),
    "scale": dict(scale=float("nan")),
}


@pytest.mark.parametrize("what", BAD)
@pytest.mark.parametrize("call", [forward, backward])
def test_refused(call, what):
    with pytest.raises(ValueError):
        call(**BAD[what])


MORE = {
    "result of another shape": (forward, dict(out=rows(H * D, n=T + 1))),
    "result in fp32": (forward, dict(out=rows(H * D, torch.float32))),
    "lse in bf16": (forward, dict(lse=torch.zeros(W, H, HIGH * WIDE).to(BF))),
    "gradient of another shape": (backward, dict(d_o=rows(H * D + 1))),
    "lse of another shape": (backward, dict(lse=torch.zeros(W, HIGH * WIDE, H))),
    "place of another shape": (backward, dict(dqkv=rows(H * D))),
    "table gradient in bf16": (backward, dict(dtable=torch.zeros(OFF, H).to(BF))),
    "table gradient that is not wanted": (backward, dict(dtable=torch.zeros(OFF, H), need_dtable=False)),
}


@pytest.mark.parametrize("what", MORE)
def test_refused_by_one(what):
    call, over = MORE[what]
    with pytest.raises(ValueError):
        call(**over)


def test_results_over_other_tensors_are_refused():
    both = rows(4 * H * D)
    with pytest.raises(ValueError, match="lies over"):
        forward(qkv=both[:, :3 * H * D], out=both[:, 2 * H * D:3 * H * D])
    qkv = rows(3 * H * D)
    with pytest.raises(ValueError, match="lies over"):
        backward(qkv=qkv, dqkv=qkv)
    table = torch.zeros(OFF, H)
    with pytest.raises(ValueError, match="lies over"):
        backward(table=table, dtable=table)


def test_cpu_tensors_are_refused_and_not_computed_elsewhere():
    with pytest.raises(ValueError, match="GPU"):
        forward()
    with pytest.raises(ValueError, match="GPU"):
        backward()


def test_relative_positions():
    assert PB.relative_positions((1, 1)) == 1 and PB.relative_positions((HIGH, WIDE)) == OFF
