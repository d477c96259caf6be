"""Refusals of layer norm: made on the host, before anything is launched."""
import pytest
import torch

from aeris_gb_b200.ops import layer_norm as LN

ROWS, COLS = 6, 32


def mat(rows=ROWS, cols=COLS, dt=torch.float32):
    return torch.randn(rows, cols).to(dt)


FORWARD = {
    "three dimensions": dict(x=torch.randn(2, 3, 4)),
    "half": dict(x=mat().half()),
    "no columns": dict(x=mat(3, 0)),
    "columns apart": dict(x=mat(COLS, ROWS).t()),
    "weight of another width": dict(weight=torch.ones(COLS + 1)),
    "weight in half": dict(weight=torch.ones(COLS).half()),
    "weight with gaps": dict(weight=torch.ones(2 * COLS)[::2]),
    "types differ": dict(weight=torch.ones(COLS), bias=torch.ones(COLS).bfloat16()),
    "result of another shape": dict(out=mat(ROWS + 1)),
    "result of another type": dict(out=mat(dt=torch.bfloat16)),
    "expanded result": dict(out=torch.empty(1, COLS).expand(ROWS, COLS)),
    "result over itself": dict(out=torch.empty(ROWS * COLS).as_strided((ROWS, COLS), (COLS // 2, 1))),
    "statistics in bf16": dict(stats=torch.empty(ROWS, 2).bfloat16()),
    "statistics of another shape": dict(stats=torch.empty(ROWS, 3)),
}


@pytest.mark.parametrize("what", FORWARD)
def test_forward_refused(what):
    a = dict(x=mat(), weight=None, bias=None, out=None, stats=None)
    a.update(FORWARD[what])
    with pytest.raises(ValueError):
        LN.layer_norm_fwd(a["x"], a["weight"], a["bias"], eps=1e-5, out=a["out"], stats=a["stats"])


def test_results_beside_their_input_are_refused():
    wide = torch.randn(ROWS + 1, COLS)
    with pytest.raises(ValueError, match="beside"):
        LN.layer_norm_fwd(wide[:-1], eps=1e-5, out=wide[1:])
    with pytest.raises(ValueError, match="beside"):
        LN.layer_norm_bwd(wide[:-1], mat(), torch.empty(ROWS, 2), dx=wide[1:])
    flat = torch.randn(ROWS * COLS)
    with pytest.raises(ValueError, match="stats"):
        LN.layer_norm_fwd(flat.view(ROWS, COLS), eps=1e-5, stats=flat[:2 * ROWS].view(ROWS, 2))


BACKWARD = {
    "dy of another shape": dict(dy=mat(ROWS + 1)),
    "dy of another type": dict(dy=mat(dt=torch.bfloat16)),
    "statistics of other rows": dict(stats=torch.empty(ROWS + 1, 2)),
    "dw without a weight": dict(weight=None, dw=torch.zeros(COLS)),
    "dw alone": dict(dw=torch.zeros(COLS)),
    "db without a bias": dict(bias=False, dw=torch.zeros(COLS), db=torch.zeros(COLS)),
    "dw in bf16": dict(dw=torch.zeros(COLS).bfloat16(), db=torch.zeros(COLS)),
    "dw of another width": dict(dw=torch.zeros(COLS + 1), db=torch.zeros(COLS)),
}


@pytest.mark.parametrize("what", BACKWARD)
def test_backward_refused(what):
    a = dict(dy=mat(), x=mat(), stats=torch.empty(ROWS, 2), weight=torch.ones(COLS), bias=True, dw=None, db=None)
    a.update(BACKWARD[what])
    with pytest.raises(ValueError):
        LN.layer_norm_bwd(a["dy"], a["x"], a["stats"], a["weight"], bias=a["bias"], dw=a["dw"], db=a["db"])


def test_one_place_for_both_sums_is_refused():
    t = torch.zeros(COLS)
    with pytest.raises(ValueError, match="same memory"):
        LN.layer_norm_bwd(mat(), mat(), torch.empty(ROWS, 2), torch.ones(COLS), dw=t, db=t)


def test_cpu_tensors_are_refused_and_not_computed_elsewhere():
    with pytest.raises(ValueError, match="GPU"):
        LN.layer_norm_fwd(mat(), eps=1e-5)
    with pytest.raises(ValueError, match="GPU"):
        LN.layer_norm_bwd(mat(), mat(), torch.empty(ROWS, 2))


def test_slices_cover_the_rows_and_the_machine():
    for rows, cols in ((1, 1), (5, 20000), (64800, 1536), (2 ** 31 - 1, 1)):
        s = LN.slices_for(rows, cols, 148)
        assert s <= 65535 and (s == 1) == (rows * cols <= 2 ** 14 and cols <= 4096)


@pytest.mark.parametrize("start", [1, 3])
def test_statistics_between_8_byte_boundaries_are_refused(start):
    flat = torch.zeros(2 * ROWS + 4)
    stats = flat[start:start + 2 * ROWS].view(ROWS, 2)
    assert stats.is_contiguous() and stats.data_ptr() % 8 == 4
    with pytest.raises(ValueError, match="8-byte"):
        LN.layer_norm_fwd(mat(), eps=1e-5, stats=stats)
    with pytest.raises(ValueError, match="8-byte"):
        LN.layer_norm_bwd(mat(), mat(), stats)
    with pytest.raises(ValueError, match="GPU"):          # two further on: taken
        LN.layer_norm_bwd(mat(), mat(), flat[2:2 + 2 * ROWS].view(ROWS, 2))


@pytest.mark.parametrize("rows,cols,slices", [
    (1, 1, 1), (256, 256, 1), (256, 257, 64), (257, 8, 65), (250, 200, 1), (1000, 10, 250), (16, 4096, 1), (17, 4096, 5), (15, 4097, 15),
    (1, 4097, 2), (2368, 64, 592), (2369, 64, 592), (147, 16384, 147), (149, 16384, 148), (64800, 1536, 592), (1000, 10 ** 6, 148), (2, 2 ** 31 - 2 ** 10, 2)])
def test_slices_of_the_rows(rows, cols, slices):
    """One (a cluster's) up to 256 rows and 2^16 elements of rows of up to 4,096; at most four a multiprocessor, of four rows; of
    wider rows one a multiprocessor, of one row. Two at least where there is a workspace."""
    assert LN.slices_for(rows, cols, 148) == slices
