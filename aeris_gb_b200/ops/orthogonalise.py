"""Python front ends of the orthogonalisation of matrices and of the optimizer step that uses it (``csrc/orthogonalise.cu``).

    X = U / max(|U|_F, eps);   X <- a X + (b S + c S^2) X,  S = X X^T      ``steps`` times, (a, b, c) = COEFFICIENTS

replaces the singular values of U by values around 1 (0.68 to 1.2 after five steps, for those above 1 % of the norm) and keeps its
singular vectors.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import lib as _l

_P, _I, _F, _LL, _D = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong, ctypes.c_double
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_COUNT = 65535            # matrices per launch: one layer of the grid each
PARTS = 128                  # partial sums of squares per matrix
# Workspace of one batch; what does not fit goes in several.
WORKSPACE_BYTES = 1 << 30


class _In(ctypes.Structure):
    """Mirror of ``AerisOrthoIn`` (csrc/api.h)."""
    _fields_ = ([(n, _P) for n in ("x", "grad", "momentum", "norm_sq", "offsets", "X", "partial", "status")] + [("eps", _D)]
                + [(n, _LL) for n in ("stride", "numel")]
                + [(n, _I) for n in ("rows", "cols", "ld", "count", "behind", "bf16", "nesterov", "zero_grad")]
                + [(n, _F) for n in ("beta", "grad_scale", "max_norm")])


class _Out(ctypes.Structure):
    """Mirror of ``AerisOrthoOut`` (csrc/api.h)."""
    _fields_ = ([(n, _P) for n in ("X", "out", "master", "ema", "weights", "offsets", "status")]
                + [(n, _LL) for n in ("stride", "numel")] + [(n, _I) for n in ("rows", "cols", "ld", "count", "behind")]
                + [(n, _F) for n in ("decay", "rate", "ema_beta")])


def _pitch(n: int) -> int:
    return -(-n // 64) * 64


class _Batch:
    """Workspaces of ``count`` matrices of shorter side ``d`` and longer side ``k``, and the products on them."""

    def __init__(self, count: int, d: int, k: int, steps: int, device):
        self.count, self.d, self.k, self.steps = count, d, k, steps
        self.x_size, self.half = d * _pitch(k), count * d * _pitch(k)
        s = _l.lib().aeris_ortho_buffers(d, k, steps) * count * d * _pitch(d)
        self.x = torch.empty(2 * self.half, dtype=torch.float16, device=device)
        self.s = torch.empty(s, dtype=torch.float16, device=device)
        self.partial = torch.empty(count * PARTS, dtype=torch.float64, device=device)

    @staticmethod
    def most(d: int, k: int, steps: int) -> int:
        """Matrices of one batch."""
        per = 2 * (2 * d * _pitch(k) + _l.lib().aeris_ortho_buffers(d, k, steps) * d * _pitch(d))
        return max(1, min(MAX_COUNT, WORKSPACE_BYTES // per))

    def load(self, first: int, a: _In) -> None:
        a.X, a.partial = self.x.data_ptr() + 2 * first * self.x_size, self.partial.data_ptr()
        _l.check(_l.lib().aeris_ortho_in(ctypes.byref(a), _l.stream_ptr()), "aeris_ortho_in", kernels=2)

    def iterate(self) -> None:
        """Leaves the result in ``self.result``."""
        lib = _l.lib()
        rc = lib.aeris_ortho_iterate(_l.ptr(self.x), _l.ptr(self.s), self.count, self.d, self.k, self.steps,
                                     _l.ptr(_l.status_word()), _l.stream_ptr())
        _l.check(min(rc, 0), "aeris_ortho_iterate", kernels=max(rc, 0))
        self.result = self.x.data_ptr() + 2 * self.half * (lib.aeris_ortho_updates(self.d, self.k, self.steps) & 1)

    def store(self, first: int, a: _Out) -> None:
        a.X = self.result + 2 * first * self.x_size
        _l.check(_l.lib().aeris_ortho_out(ctypes.byref(a), _l.stream_ptr()), "aeris_ortho_out")


def _as_batch(t: torch.Tensor) -> torch.Tensor:
    return t.unsqueeze(0) if t.dim() == 2 else t


def _pitched(t: torch.Tensor) -> bool:
    """Whether the kernels find the elements of ``t`` [count, rows, cols]: columns side by side, rows one behind the other."""
    return (t.stride(2) == 1 or t.shape[2] == 1) and (t.shape[1] == 1 or t.stride(1) >= t.shape[2])


def _row_pitch(t: torch.Tensor) -> int:
    return t.stride(1) if t.shape[1] > 1 else t.shape[2]


def _check_steps(steps: int) -> None:
    if not isinstance(steps, int) or not 1 <= steps <= 20:
        raise ValueError(f"1 to 20 steps are taken, got {steps!r}")


def orthogonalise(x: torch.Tensor, *, steps: int = 5, eps: float = 1e-7, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x`` [rows, cols] or [count, rows, cols], fp32 or bf16, each matrix by itself; bf16 result of the same shape, ``out``
    where given (any pitch between rows; may not share memory with ``x``). A matrix of zeros stays one; one that holds a NaN or
    an infinity becomes NaN, the others of its batch do not notice."""
    _check_steps(steps)
    if x.dim() not in (2, 3) or x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"fp32 or bf16 [rows, cols] or [count, rows, cols], got {x.dtype} {tuple(x.shape)}")
    if out is not None:
        o = _as_batch(out)
        if out.shape != x.shape or out.dtype != torch.bfloat16 or out.device != x.device or (out.numel() and not (
                _pitched(o) and (o.shape[0] == 1 or o.stride(0) >= (o.shape[1] - 1) * _row_pitch(o) + o.shape[2]))):
            raise ValueError(f"out: bf16 {tuple(x.shape)} on {x.device} whose rows do not overlap, got {out.dtype} "
                             f"{tuple(out.shape)} on {out.device} with strides {out.stride()}")
    _l.require_cuda(x)
    if out is None:
        out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    if x.numel() == 0:
        return out
    xs, os = _as_batch(x.detach()), _as_batch(out)
    if not _pitched(xs):
        xs = xs.contiguous()
    count, rows, cols = xs.shape
    d, k = min(rows, cols), max(rows, cols)
    with _l.on_device(x.device):
        status = _l.status_word().data_ptr()
        most = _Batch.most(d, k, steps)
        for i in range(0, count, most):
            n = min(most, count - i)
            b = _Batch(n, d, k, steps, x.device)
            a = _In(x=xs.data_ptr() + i * xs.stride(0) * xs.element_size(), bf16=xs.dtype == torch.bfloat16, stride=xs.stride(0),
                    rows=rows, cols=cols, ld=_row_pitch(xs), count=n, eps=eps, status=status)
            b.load(0, a)
            b.iterate()
            b.store(0, _Out(out=os.data_ptr() + i * os.stride(0) * 2, stride=os.stride(0), rows=rows, cols=cols,
                            ld=_row_pitch(os), count=n, status=status))
    return out


def _check_flat(name: str, t: torch.Tensor, like: torch.Tensor, dtype: torch.dtype) -> None:
    if t.dim() != 1 or t.shape != like.shape or t.dtype != dtype or t.device != like.device or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype} [{like.numel()}] on {like.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.data_ptr() % 16:
        raise ValueError(f"{name} does not start on a 16-byte boundary")


def _step_batches(d, k, parts, master, grad, momentum, weights, ema, norm_sq, status, steps, settings, rates) -> None:
    """All matrices of sides ``d`` and ``k``, upright and wide ones in the same products, as many at a time as fit a batch."""
    todo = [(rows, cols, off.data_ptr(), 0, off.numel()) for rows, cols, off in parts]
    left, most = sum(n for *_, n in todo), _Batch.most(d, k, steps)
    batch, taken = None, []
    while left:
        if batch is None:
            batch, room = _Batch(min(most, left), d, k, steps, master.device), min(most, left)
            first, taken = 0, []
        rows, cols, table, start, n = todo.pop(0)
        m = min(n, room)
        at = dict(offsets=table + 8 * start, behind=start > 0, numel=master.numel(), rows=rows, cols=cols, ld=cols, count=m,
                  status=status)
        batch.load(first, _In(grad=grad.data_ptr(), momentum=momentum.data_ptr(),
                              norm_sq=0 if norm_sq is None else norm_sq.data_ptr(), **at, **settings))
        taken.append((first, at))
        first, room, left = first + m, room - m, left - m
        if m < n:
            todo.insert(0, (rows, cols, table, start + m, n - m))
        if not room:
            batch.iterate()
            for i, where in taken:
                batch.store(i, _Out(master=master.data_ptr(), weights=0 if weights is None else weights.data_ptr(),
                                    ema=0 if ema is None else ema.data_ptr(), **where, **rates))
            batch = None


def orthogonal_step(master: torch.Tensor, grad: torch.Tensor, momentum: torch.Tensor, weights: torch.Tensor | None,
                    ema: torch.Tensor | None, norm_sq: torch.Tensor | None, *, groups, lr: float, beta: float, nesterov: bool,
                    weight_decay: float, scale: float, grad_scale: float, max_norm: float, ema_beta: float, steps: int = 5,
                    eps: float = 1e-7, zero_grad: bool = True) -> None:
    """One optimizer step of the matrices of flat fp32 buffers, counterpart of :func:`.elementwise.adamw`::

        g = nan_to_num(grad * grad_scale * clip);  M = beta M + (1 - beta) g;  U = beta M + (1 - beta) g  (nesterov)  or  M
        master = master (1 - lr weight_decay) - lr scale sqrt(max(rows, cols)) orthogonalise(U)

    ``weights`` (bf16) receives the new master, ``ema`` its running average (``ema_beta`` < 0: not), ``grad`` zeros with
    ``zero_grad``. ``norm_sq`` and ``max_norm``: clipping as in ``adamw``. ``groups``: (rows, cols, offsets) for matrices that lie
    without gaps from the element offsets on, an int64 tensor on the same device, ascending; no two matrices may overlap. One
    that does not lie inside the buffers, or not behind the one before it, sets the status word and is left as it is; elements
    of no matrix are not touched. ``scale`` = 0.2 gives updates the root mean square of AdamW's."""
    _check_steps(steps)
    if master.dim() != 1 or master.dtype != torch.float32 or not master.is_contiguous() or master.data_ptr() % 16:
        raise ValueError(f"master: contiguous fp32 [n] from a 16-byte boundary on, got {master.dtype} {tuple(master.shape)}")
    for name, t, dt in (("grad", grad, torch.float32), ("momentum", momentum, torch.float32), ("weights", weights, torch.bfloat16),
                        ("ema", ema, torch.float32)):
        if t is not None:
            _check_flat(name, t, master, dt)
    if norm_sq is not None and (norm_sq.numel() != 1 or norm_sq.dtype != torch.float64 or norm_sq.device != master.device):
        raise ValueError(f"norm_sq: one fp64 value on {master.device}, got {norm_sq.dtype} {tuple(norm_sq.shape)}")
    batches: dict[tuple[int, int], list] = {}
    for rows, cols, offsets in groups:
        if rows < 1 or cols < 1 or offsets.dim() != 1 or offsets.dtype != torch.int64 or offsets.device != master.device \
                or not offsets.is_contiguous():
            raise ValueError(f"groups hold (rows, cols, contiguous int64 offsets on {master.device}), got ({rows}, {cols}, "
                             f"{offsets.dtype} {tuple(offsets.shape)} on {offsets.device})")
        if rows * cols * offsets.numel() > master.numel():
            raise ValueError(f"{offsets.numel()} matrices of {rows} x {cols} do not fit {master.numel()} elements")
        if offsets.numel():
            batches.setdefault((min(rows, cols), max(rows, cols)), []).append((rows, cols, offsets))
    _l.require_cuda(master)
    with _l.on_device(master.device):
        status = _l.status_word().data_ptr()
        for (d, k), parts in batches.items():
            _step_batches(d, k, parts, master, grad, momentum, weights, ema, norm_sq, status, steps,
                          dict(beta=beta, nesterov=nesterov, zero_grad=zero_grad, grad_scale=grad_scale, max_norm=max_norm, eps=eps),
                          dict(decay=1.0 - lr * weight_decay, rate=lr * scale * math.sqrt(k), ema_beta=ema_beta))
