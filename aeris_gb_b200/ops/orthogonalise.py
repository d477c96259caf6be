"""Python front ends of the orthogonalisation of matrices and of the optimizer step that uses it (``csrc/orthogonalise.cu``).

    X = U / max(|U|_F, eps);   X <- a X + (b S + c S^2) X,  S = X X^T      ``steps`` times, (a, b, c) = COEFFICIENTS

replaces the singular values of U by values around 1 (0.68 to 1.2 after five steps, for those above 1 % of the norm) and keeps its
singular vectors. Products take fp16 operands and sum in fp32: a result is about 1e-3 of its norm off before it is rounded, 1e-2 where a
matrix has a low rank, an eighth to a twelfth of what bf16 operands leave. The same call gives the same bits; which other matrices
share it can change the last ones.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct

import torch

from . import lib as _l

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_GROUPS, MAX_LENGTHS = 4, 2       # shapes of a batch, and longer sides among them
MAX_SIDE = 1 << 30                   # rows or columns of a matrix
MIN_EPS = 1e-30                      # one over it, times the scale of the fp16 factors, is a 32-bit number
MAX_COUNT = 1 << 16                  # matrices of a group
FEW_ROWS, SHORT_ROWS = 128, 384      # up to so many rows (d) matrices with rows longer than that have a batch for each length
WORKSPACE_BYTES = 1 << 30            # of one batch; what does not fit goes in several

# AerisOrthoGroup and AerisOrtho (csrc/api.h), field by field
_GROUP = struct.Struct("Pqq6if4x")
_REST = struct.Struct("10Pdqq5i5f")


def _group(rows, cols, count, *, offsets=0, stride=0, out_stride=0, ld=0, ld_out=0, behind=False, rate=0.0) -> bytes:
    return _GROUP.pack(offsets, stride, out_stride, rows, cols, ld or cols, ld_out, count, behind, rate)


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    f = getattr(_l.lib(), name)
    if name == "aeris_ortho_work_bytes":
        f.argtypes, f.restype = (ctypes.c_char_p,), ctypes.c_longlong
    elif name == "aeris_ortho_route":
        f.argtypes = (ctypes.c_char_p,)
    else:
        f.argtypes = (ctypes.c_char_p, ctypes.c_void_p)
    return f


@functools.lru_cache(maxsize=4096)
def _work_bytes(shapes: tuple, steps: int) -> int:
    """Workspace of a batch of (rows, cols, how many)."""
    n = _entry("aeris_ortho_work_bytes")(_shapes_alone(shapes, steps))
    _l.check(min(n, 0), "aeris_ortho_work_bytes", kernels=0)
    return n


def _shapes_alone(shapes: tuple, steps: int) -> bytes:
    rest = _REST.pack(*[0] * 10, 0.0, 0, 0, len(shapes), steps, 0, 0, 0, *[0.0] * 5)
    return b"".join(_group(*g) for g in shapes) + bytes(_GROUP.size * (MAX_GROUPS - len(shapes))) + rest


_ROUTES = ("one launch", "gram alone", "two steps", "gram parts", "gram pairs", "factor pairs", "update pairs")


def route(shapes, steps: int = 5) -> set[str]:
    """How a batch of (rows, cols, how many) with one shorter side goes on the current device (``ORTHO_ROUTE_``* of csrc/api.h)."""
    rc = _entry("aeris_ortho_route")(_shapes_alone(tuple(shapes), steps))
    _l.check(min(rc, 0), "aeris_ortho_route", kernels=0)
    return {name for i, name in enumerate(_ROUTES) if rc >> i & 1}


def _bytes_per_matrix(d: int, k: int) -> int:
    """Workspace of one matrix, about: two X, four square factors, partial sums."""
    few = min(16, max(1, k // 512)) * 65536 if d <= FEW_ROWS and k > SHORT_ROWS else 0
    return 2 * d * (2 * (-(-k // 64) * 64) + 4 * (-(-d // 64) * 64)) + 8192 + few


def _run(device, groups: list[bytes], shapes: tuple, *, x=0, out=0, grad=0, momentum=0, master=0, ema=0, weights=0, norm_sq=0, eps,
         numel=0, steps, bf16=False, nesterov=False, zero_grad=False, beta=0.0, grad_scale=0.0, max_norm=0.0, decay=0.0,
         ema_beta=-1.0) -> None:
    n, work = _work_bytes(shapes, steps), 0
    if n:
        buf = torch.empty(n + 1024, dtype=torch.uint8, device=device)
        work = -(-buf.data_ptr() // 1024) * 1024
    rest = _REST.pack(x, out, grad, momentum, master, ema, weights, norm_sq, work, _l.status_word().data_ptr(), eps, numel, n,
                      len(groups), steps, bf16, nesterov, zero_grad, beta, grad_scale, max_norm, decay, ema_beta)
    rc = _entry("aeris_orthogonalise")(b"".join(groups) + bytes(_GROUP.size * (MAX_GROUPS - len(groups))) + rest, _l.raw_stream())
    _l.check(min(rc, 0), "aeris_orthogonalise", kernels=max(rc, 0))


def _as_batch(t: torch.Tensor) -> torch.Tensor:
    return t.unsqueeze(0) if t.dim() == 2 else t


def _pitched(t: torch.Tensor) -> bool:
    """Whether the kernels find the elements of ``t`` [count, rows, cols]: columns side by side, rows one behind the other."""
    return (t.stride(2) == 1 or t.shape[2] == 1) and (t.shape[1] == 1 or t.shape[2] <= t.stride(1) < 2 ** 31)


def _row_pitch(t: torch.Tensor) -> int:
    return t.stride(1) if t.shape[1] > 1 else t.shape[2]


def _check_steps(steps: int, eps: float) -> None:
    if not isinstance(steps, int) or not 1 <= steps <= 20:
        raise ValueError(f"1 to 20 steps are taken, got {steps!r}")
    if not MIN_EPS <= eps < math.inf:
        raise ValueError(f"eps from {MIN_EPS} on is taken, got {eps!r}")


def orthogonalise(x: torch.Tensor, *, steps: int = 5, eps: float = 1e-7, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x`` [rows, cols] or [count, rows, cols], fp32 or bf16, each matrix by itself; bf16 result of the same shape, ``out``
    where given (any pitch between rows; may not share memory with ``x``). A matrix of zeros stays one; one that holds a NaN or
    an infinity becomes NaN, the others of its batch do not notice."""
    _check_steps(steps, eps)
    if x.dim() not in (2, 3) or x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"fp32 or bf16 [rows, cols] or [count, rows, cols], got {x.dtype} {tuple(x.shape)}")
    if max(x.shape[-2:]) > MAX_SIDE:
        raise ValueError(f"matrices of up to {MAX_SIDE} rows and columns are taken, got {tuple(x.shape)}")
    if out is not None:
        o = _as_batch(out)
        if out.shape != x.shape or out.dtype != torch.bfloat16 or out.device != x.device or (out.numel() and not (
                _pitched(o) and (o.shape[0] == 1 or o.stride(0) >= (o.shape[1] - 1) * _row_pitch(o) + o.shape[2]))):
            raise ValueError(f"out: bf16 {tuple(x.shape)} on {x.device} whose rows do not overlap, got {out.dtype} "
                             f"{tuple(out.shape)} on {out.device} with strides {out.stride()}")
        if _l.share_memory(out, x):
            raise ValueError("out shares memory with x")
    _l.require_cuda(x)
    if out is None:
        out = torch.empty_like(x, dtype=torch.bfloat16, memory_format=torch.contiguous_format)
    if x.numel() == 0:
        return out
    xs, os = _as_batch(x), _as_batch(out)
    if not _pitched(xs):
        xs = xs.contiguous()
    count, rows, cols = xs.shape
    most = max(1, min(MAX_COUNT, WORKSPACE_BYTES // _bytes_per_matrix(min(rows, cols), max(rows, cols))))
    stride, out_stride, ld, ld_out = xs.stride(0), os.stride(0), _row_pitch(xs), _row_pitch(os)
    with _l.on_device(x.device):
        for i in range(0, count, most):
            n = min(most, count - i)
            _run(x.device, [_group(rows, cols, n, stride=stride, out_stride=out_stride, ld=ld, ld_out=ld_out)], ((rows, cols, n),),
                 x=xs.data_ptr() + i * stride * xs.element_size(), out=os.data_ptr() + i * out_stride * 2,
                 bf16=xs.dtype is torch.bfloat16, eps=eps, steps=steps)
    return out


def _check_flat(name: str, t: torch.Tensor, like: torch.Tensor, dtype: torch.dtype) -> None:
    if t.dim() != 1 or t.shape != like.shape or t.dtype != dtype or t.device != like.device or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype} [{like.numel()}] on {like.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.data_ptr() % 16:
        raise ValueError(f"{name} does not start on a 16-byte boundary")


def _batches(groups):
    """Cuts groups (rows, cols, address of the offsets, how many) into batches: lists of (rows, cols, address, how many, whether
    an entry of the same table lies before it) with one shorter side, at most MAX_LENGTHS longer ones, MAX_GROUPS parts and
    WORKSPACE_BYTES. Shapes with one shorter side share the launches of their square factors."""
    by_side: dict[tuple[int, int], list] = {}
    for g in groups:
        d, k = min(g[:2]), max(g[:2])
        by_side.setdefault((d, k if d <= FEW_ROWS and k > SHORT_ROWS else 0), []).append(g)
    for (d, _), todo in by_side.items():
        batch, lengths, room = [], set(), WORKSPACE_BYTES
        todo = [(*g, False) for g in todo][::-1]
        while todo:
            rows, cols, table, n, behind = todo.pop()
            k = max(rows, cols)
            per = _bytes_per_matrix(d, k)
            m = min(n, MAX_COUNT, max(room // per, 0 if batch else 1))
            if m == 0 or len(batch) == MAX_GROUPS or (k not in lengths and len(lengths) == MAX_LENGTHS):
                yield batch
                batch, lengths, room = [], set(), WORKSPACE_BYTES
                todo.append((rows, cols, table, n, behind))
                continue
            batch.append((rows, cols, table, m, behind))
            lengths.add(k)
            room -= m * per
            if m < n:
                todo.append((rows, cols, table + 8 * m, n - m, True))
        if batch:
            yield batch


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
    that does not lie inside the buffers, or not behind the one before it, is left as it is and sets the status word, and so
    does one that shares elements with a matrix of another group in the same launch (one shorter side): the call has then
    failed (``lib.check_status`` raises), and which of its other matrices have been updated is not defined. Elements of no
    matrix are not touched. ``scale`` = 0.2 gives updates the root mean square of AdamW's."""
    _check_steps(steps, eps)
    if master.dim() != 1 or master.dtype != torch.float32 or not master.is_contiguous() or master.data_ptr() % 16:
        raise ValueError(f"master: contiguous fp32 [n] from a 16-byte boundary on, got {master.dtype} {tuple(master.shape)}")
    for name, t, dt in (("grad", grad, torch.float32), ("momentum", momentum, torch.float32), ("weights", weights, torch.bfloat16),
                        ("ema", ema, torch.float32)):
        if t is not None:
            _check_flat(name, t, master, dt)
    at = sorted([t.data_ptr() for t in (master, grad, momentum, ema) if t is not None])
    size = 4 * master.numel()
    if any(b - a < size for a, b in zip(at, at[1:])) or weights is not None and any(
            -size < a - weights.data_ptr() < size // 2 for a in at):
        raise ValueError("the buffers of a step share memory")
    if norm_sq is not None and (norm_sq.numel() != 1 or norm_sq.dtype != torch.float64 or norm_sq.device != master.device):
        raise ValueError(f"norm_sq: one fp64 value on {master.device}, got {norm_sq.dtype} {tuple(norm_sq.shape)}")
    todo = []
    for rows, cols, offsets in groups:
        if not 1 <= rows <= MAX_SIDE or not 1 <= cols <= MAX_SIDE or offsets.dim() != 1 or offsets.dtype != torch.int64 or offsets.device != master.device \
                or not offsets.is_contiguous():
            raise ValueError(f"groups hold (rows, cols, contiguous int64 offsets on {master.device}), got ({rows}, {cols}, "
                             f"{offsets.dtype} {tuple(offsets.shape)} on {offsets.device})")
        if rows * cols * offsets.numel() > master.numel():
            raise ValueError(f"{offsets.numel()} matrices of {rows} x {cols} do not fit {master.numel()} elements")
        if offsets.numel():
            todo.append((rows, cols, offsets.data_ptr(), offsets.numel()))
    _l.require_cuda(master)
    with _l.on_device(master.device):
        common = dict(grad=grad.data_ptr(), momentum=momentum.data_ptr(), master=master.data_ptr(), numel=master.numel(),
                      weights=0 if weights is None else weights.data_ptr(), ema=0 if ema is None else ema.data_ptr(),
                      norm_sq=0 if norm_sq is None else norm_sq.data_ptr(), eps=eps, steps=steps, nesterov=nesterov,
                      zero_grad=zero_grad, beta=beta, grad_scale=grad_scale, max_norm=max_norm, decay=1.0 - lr * weight_decay,
                      ema_beta=ema_beta)
        for batch in _batches(todo):
            _run(master.device, [_group(rows, cols, n, offsets=table, behind=behind, rate=lr * scale * math.sqrt(max(rows, cols)))
                                 for rows, cols, table, n, behind in batch],
                 tuple((rows, cols, n) for rows, cols, _, n, _ in batch), **common)
