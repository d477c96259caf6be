"""Refusals of linear layers: made on the host, before anything is launched."""
import pytest
import torch

from aeris_gb_b200.ops import linear as LI

ROWS, INNER, COLS = 6, 16, 24
BF = torch.bfloat16


def mat(rows, cols, dt=BF):
    return torch.randn(rows, cols).to(dt)


def forward(**over):
    a = dict(x=mat(ROWS, INNER), w=mat(COLS, INNER), bias=None, act="gelu", resid=None, keep=False, out=None, z=None)
    a.update(over)
    return LI.linear_fwd(a.pop("x"), a.pop("w"), a.pop("bias"), **a)


def backward(**over):
    a = dict(dy=mat(ROWS, COLS), x=mat(ROWS, INNER), w=mat(COLS, INNER), z=mat(ROWS, COLS), act="gelu")
    a.update(over)
    return LI.linear_bwd(a.pop("dy"), a.pop("x"), a.pop("w"), a.pop("z"), **a)


FORWARD = {
    "fp32": dict(x=mat(ROWS, INNER, torch.float32)),
    "one dimension": dict(x=torch.randn(INNER).to(BF)),
    "inner sizes differ": dict(w=mat(COLS, INNER + 1)),
    "no columns": dict(w=mat(0, INNER)),
    "nothing to add up": dict(x=mat(ROWS, 0), w=mat(COLS, 0)),
    "columns apart": dict(w=mat(INNER, COLS).t()),
    "bias of another width": dict(bias=torch.zeros(COLS + 1)),
    "bias in half": dict(bias=torch.zeros(COLS).half()),
    "bias with gaps": dict(bias=torch.zeros(2 * COLS)[::2]),
    "unknown activation": dict(act="mish"),
    "residual of another shape": dict(resid=mat(ROWS, COLS + 1)),
    "residual in fp32": dict(resid=mat(ROWS, COLS, torch.float32)),
    "result of another shape": dict(out=mat(ROWS + 1, COLS)),
    "result in fp32": dict(out=mat(ROWS, COLS, torch.float32)),
    "expanded result": dict(out=mat(1, COLS).expand(ROWS, COLS)),
    "z without keep": dict(z=mat(ROWS, COLS)),
    "z of another shape": dict(keep=True, z=mat(ROWS, COLS + 1)),
}


@pytest.mark.parametrize("what", FORWARD)
def test_forward_refused(what):
    with pytest.raises(ValueError):
        forward(**FORWARD[what])


def test_results_over_other_tensors_are_refused():
    wide = mat(2 * ROWS, COLS)
    with pytest.raises(ValueError, match="lies over"):
        forward(resid=wide[1:ROWS + 1], out=wide[:ROWS])
    with pytest.raises(ValueError, match="lies over"):
        forward(keep=True, out=wide[:ROWS], z=wide[:ROWS])
    square = mat(ROWS, INNER)
    with pytest.raises(ValueError, match="lies over"):
        forward(x=square, w=mat(INNER, INNER), out=square)
    with pytest.raises(ValueError, match="lies over"):
        backward(x=square, w=mat(INNER, INNER), dy=mat(ROWS, INNER), z=mat(ROWS, INNER), dx=square)


BACKWARD = {
    "no z": dict(z=None),
    "z of another shape": dict(z=mat(ROWS, COLS + 1)),
    "z in fp32": dict(z=mat(ROWS, COLS, torch.float32)),
    "dy of another shape": dict(dy=mat(ROWS + 1, COLS)),
    "unknown activation": dict(act=None),
    "a place for dx that is not wanted": dict(need_dx=False, dx=mat(ROWS, INNER)),
    "a place for db that is not wanted": dict(bias=False, db=torch.zeros(COLS)),
    "dw in bf16": dict(dw=mat(COLS, INNER)),
    "db in bf16": dict(db=torch.zeros(COLS, dtype=BF)),
    "dw of another shape": dict(dw=mat(COLS + 1, INNER, torch.float32)),
    "dx in fp32": dict(dx=mat(ROWS, INNER, torch.float32)),
}


@pytest.mark.parametrize("what", BACKWARD)
def test_backward_refused(what):
    with pytest.raises(ValueError):
        backward(**BACKWARD[what])


def test_cpu_tensors_are_refused_and_not_computed_elsewhere():
    with pytest.raises(ValueError, match="GPU"):
        forward()
    with pytest.raises(ValueError, match="GPU"):
        backward()



def test_a_result_over_an_operand_is_refused_where_that_is_the_residual_too():
    """Rows of x are read by blocks that make other columns of the result."""
    square, w = mat(INNER, INNER), mat(INNER, INNER)
    with pytest.raises(ValueError, match="lies over"):
        forward(x=square, w=w, resid=square, out=square)
    with pytest.raises(ValueError, match="lies over"):
        forward(x=square, w=w, resid=square, out=square[:])
    with pytest.raises(ValueError, match="lies over"):
        forward(x=square, w=w, resid=w, out=w)
    with pytest.raises(ValueError, match="lies over"):
        forward(x=square, w=w, keep=True, resid=square, z=square)
    with pytest.raises(ValueError, match="GPU"):          # a residual of its own
        other = mat(INNER, INNER)
        forward(x=square, w=w, resid=other, out=other)
    with pytest.raises(ValueError, match="GPU"):          # x is the residual, the result lies elsewhere
        forward(x=square, w=w, resid=square, out=mat(INNER, INNER))
