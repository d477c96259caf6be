"""The block of a plain window transformer out of its operators: x2 = x + proj(attention(norm(x))), out = x2 + fc2(gelu(fc1(norm(x2)))),
with a learned position bias in the attention, forward and backward, against its formulas and their derivatives in 64 bits.

Tolerance. Every tensor that the operators round to bf16 is off by at most 2^-8 of each value. The same formulas with every one of these
values (and, on the way back, every such gradient) multiplied by 1 + 2^-8 or 1 - 2^-8 at random move the results by as much as
independent roundings of that size do, in the 2-norm; real ones are at most that, and by their root mean square 1 / sqrt(3) of
it. What fp32 adds is 2^-15 of that."""
import pytest
import torch

from aeris_gb_b200.ops import layer_norm as LN
from aeris_gb_b200.ops import linear as LI
from aeris_gb_b200.ops import position_bias as PB

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
HALF = 2.0 ** -8
EPS = 1e-5
SHAPES = [(1, (1, 1), 1, 8, 16), (6, (8, 8), 4, 32, 512), (3, (5, 7), 3, 24, 200), (2, (12, 16), 2, 64, 384), (2, (15, 20), 4, 128, 1024),
          (40, (8, 8), 3, 72, 864)]
NAMES = ("out", "dx", "norm1.w", "norm1.b", "qkv.w", "qkv.b", "table", "proj.w", "proj.b", "norm2.w", "norm2.b", "fc1.w", "fc1.b",
         "fc2.w", "fc2.b")


def make(n_win, window, heads, d, hidden, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows, dim = n_win * window[0] * window[1], heads * d

    def r(*shape, size=1.0, dt=BF):
        return (torch.randn(*shape, generator=g, device=DEV) * size).to(dt)

    p = {"norm1.w": 1 + r(dim, size=0.1), "norm1.b": r(dim, size=0.1), "qkv.w": r(3 * dim, dim, size=dim ** -0.5),
         "qkv.b": r(3 * dim, size=0.1), "table": r(PB.relative_positions(window), heads, size=0.5, dt=torch.float32),
         "proj.w": r(dim, dim, size=dim ** -0.5), "proj.b": r(dim, size=0.1), "norm2.w": 1 + r(dim, size=0.1),
         "norm2.b": r(dim, size=0.1), "fc1.w": r(hidden, dim, size=dim ** -0.5), "fc1.b": r(hidden, size=0.1),
         "fc2.w": r(dim, hidden, size=hidden ** -0.5), "fc2.b": r(dim, size=0.1)}
    return p, r(rows, dim), r(rows, dim)


def block(p, x, dout, n_win, window, heads, d):
    """What a training step does with the operators; results in the order of NAMES."""
    at = (n_win, window, heads, d)
    y1, s1 = LN.layer_norm_fwd(x, p["norm1.w"], p["norm1.b"], eps=EPS)
    qkv, _ = LI.linear_fwd(y1, p["qkv.w"], p["qkv.b"])
    o, lse = PB.biased_attn_fwd(qkv, *at, p["table"])
    x2, _ = LI.linear_fwd(o, p["proj.w"], p["proj.b"], resid=x)
    y2, s2 = LN.layer_norm_fwd(x2, p["norm2.w"], p["norm2.b"], eps=EPS)
    h, z = LI.linear_fwd(y2, p["fc1.w"], p["fc1.b"], act="gelu", keep=True)
    out, _ = LI.linear_fwd(h, p["fc2.w"], p["fc2.b"], resid=x2)
    dh, dw2, db2 = LI.linear_bwd(dout, h, p["fc2.w"])
    dy2, dw1, db1 = LI.linear_bwd(dh, y2, p["fc1.w"], z, act="gelu")
    dx2, dn2w, dn2b = LN.layer_norm_bwd(dy2, x2, s2, p["norm2.w"])
    dx2 += dout
    do, dwp, dbp = LI.linear_bwd(dx2, o, p["proj.w"])
    dqkv, dtable = PB.biased_attn_bwd(do, qkv, o, lse, *at, p["table"])
    dy1, dwq, dbq = LI.linear_bwd(dqkv, y1, p["qkv.w"])
    dx, dn1w, dn1b = LN.layer_norm_bwd(dy1, x, s1, p["norm1.w"])
    dx += dx2
    return out, dx, dn1w, dn1b, dwq, dbq, dtable, dwp, dbp, dn2w, dn2b, dw1, db1, dw2, db2


class Rounded(torch.autograd.Function):
    """Moves every value by +- size of itself, and every gradient on the way back by +- back."""

    @staticmethod
    def forward(ctx, t, size, back):
        ctx.back = back
        return moved(t, size)

    @staticmethod
    def backward(ctx, g):
        return moved(g, ctx.back), None, None


def moved(t, size):
    return t * (1 + size * (2 * torch.randint(0, 2, t.shape, device=t.device) - 1)) if size else t


def formulas(p, x, dout, n_win, window, heads, d, size):
    leaf = {k: v.double().requires_grad_() for k, v in p.items()}
    x = x.double().requires_grad_()
    tokens, dim = window[0] * window[1], heads * d

    def rounded(t):
        return Rounded.apply(t, size, size)

    def norm(t, name):
        return rounded(torch.nn.functional.layer_norm(t, (dim,), leaf[name + ".w"], leaf[name + ".b"], EPS))

    def linear(t, name):
        return t @ Rounded.apply(leaf[name + ".w"], 0, size).T + leaf[name + ".b"]

    t = torch.arange(tokens, device=DEV)
    yy, xx = t // window[1], t % window[1]
    index = (yy[:, None] - yy + window[0] - 1) * (2 * window[1] - 1) + xx[:, None] - xx + window[1] - 1
    xr = Rounded.apply(x, 0, size)
    q, k, v = rounded(linear(norm(xr, "norm1"), "qkv")).reshape(n_win, tokens, 3, heads, d).permute(2, 0, 3, 1, 4)
    s = d ** -0.5 * (q @ k.transpose(-1, -2)) + leaf["table"][index].permute(2, 0, 1)
    prob = Rounded.apply(Rounded.apply(s, 0, size).softmax(-1), size, 0)
    # gradients of the product with the probabilities pass a rounding of theirs on the side of v alone
    o = rounded((prob @ v).transpose(1, 2).reshape(-1, dim))
    x2 = rounded(xr + linear(o, "proj"))
    h = rounded(torch.nn.functional.gelu(rounded(linear(norm(x2, "norm2"), "fc1"))))
    out = Rounded.apply(x2 + linear(h, "fc2"), size, 0)
    return (out.detach(), *torch.autograd.grad(out, [x, *leaf.values()], dout.double()))


@pytest.mark.parametrize("n_win,window,heads,d,hidden", SHAPES)
def test_forward_and_backward(n_win, window, heads, d, hidden):
    torch.manual_seed(0)
    p, x, dout = make(n_win, window, heads, d, hidden)
    got = block(p, x, dout, n_win, window, heads, d)
    exact = formulas(p, x, dout, n_win, window, heads, d, 0)
    off = formulas(p, x, dout, n_win, window, heads, d, HALF)
    for name, a, e, m in zip(NAMES, got, exact, off):
        bound = (m - e).norm() * (1 + 2.0 ** -6) + 2.0 ** -20 * e.norm()
        if x.numel() < 2 ** 10:
            bound = 4 * bound           # few values: their sum may come together by chance, and that of the moved ones apart
        assert (a.double() - e).norm() <= bound, (name, ((a.double() - e).norm() / e.norm()).item(), (bound / e.norm()).item())


def test_captured_and_two_at_once():
    """A step captured into a graph, the same step with other data on another stream meanwhile, and both again one after the other: the
    same bits."""
    at = (6, (8, 8), 4, 32)
    sets = [make(*at, 512, seed=i) for i in range(2)]
    want = [block(*s, *at) for s in sets]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = block(*sets[0], *at)
    for _ in range(3):
        for t in held:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = block(*sets[1], *at)
        torch.cuda.synchronize()
        for a, b in zip(held, want[0]):
            assert torch.equal(a, b)
        for a, b in zip(other, want[1]):
            assert torch.equal(a, b)


def test_two_graphs_at_once():
    """Two graphs of the same step, whose workspaces are their own, replayed beside one another."""
    at = (20, (15, 20), 2, 64)
    sets = [make(*at, 256, seed=i) for i in range(2)]
    want = [block(*s, *at) for s in sets]
    torch.cuda.synchronize()
    graphs, held = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(block(*s, *at))
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, h in zip(want, held):
        for a, b in zip(h, w):
            assert torch.equal(a, b)
