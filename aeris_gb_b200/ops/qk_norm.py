"""Python front ends of the norms of queries and keys by head with the position rotation (``csrc/qk_norm.cu``).

    z = w * x / sqrt(mean(x^2) + eps)          over the channels of one head, ``w`` shared by the heads
    y[2i], y[2i + 1] = z turned by the angle of (position, i)

The convention of :func:`.elementwise.rope_qk_`: neighbouring channels form a pair, ``cos`` / ``sin`` [L, rot / 2] fp32 hold the
angles of every position, row r of a window-major stream is at position r mod L unless ``positions`` says otherwise.
"""
from __future__ import annotations

import ctypes

import torch

from . import lib as _l

_P, _I, _LL = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
MAX_HEAD_DIM = 256


class _Heads(ctypes.Structure):
    """Mirror of ``AerisHeads`` (csrc/api.h)."""
    _fields_ = [("ptr", _P), ("row", _LL), ("head", _LL)]


class _Args(ctypes.Structure):
    """Mirror of ``AerisQkNorm`` (csrc/api.h)."""
    _fields_ = ([(n, _Heads) for n in ("q", "k", "dq", "dk", "q_out", "k_out")]
                + [(n, _P) for n in ("wq", "wk", "cos", "sin", "pos", "dwq", "dwk", "sums", "status")] + [("rows", _LL)]
                + [(n, _I) for n in ("L", "heads", "kv_heads", "d", "rot", "f32", "w_bf16", "pos64", "add_dw", "sum_rows")]
                + [("eps", ctypes.c_float)])


def _heads(t: torch.Tensor) -> _Heads:
    return _Heads(t.data_ptr(), t.stride(0), t.stride(1))


def _check_rows(name: str, t: torch.Tensor, like: torch.Tensor) -> None:
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device or (t.stride(2) != 1 and t.shape[2] > 1):
        raise ValueError(f"{name}: {tuple(t.shape)} {t.dtype} on {t.device} with strides {t.stride()}, not "
                         f"{tuple(like.shape)} {like.dtype} on {like.device} with channels side by side")


def _writable(name: str, t: torch.Tensor) -> None:
    """Refuses results of which two elements share an address (expanded rows or heads): several warps would write them."""
    (rows, heads, d), (row, head, _) = t.shape, t.stride()
    if t.numel() == 0:
        return
    by_row = (heads == 1 or head >= d) and (rows == 1 or row >= (heads - 1) * head + d)
    by_head = (rows == 1 or row >= d) and (heads == 1 or head >= (rows - 1) * row + d)
    if not (by_row or by_head):
        raise ValueError(f"{name}: elements of {tuple(t.shape)} with strides {t.stride()} share addresses")


def _prepare(q, k, wq, wk, cos, sin, eps, positions, out) -> _Args:
    """Checks that the kernels do not make, and the arguments that both directions share."""
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"q [rows, heads, d] and k [rows, kv_heads, d], got {tuple(q.shape)} and {tuple(k.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"q and k are bf16 or fp32, got {q.dtype}")
    rows, heads, d = q.shape
    if not (0 < d <= MAX_HEAD_DIM and d % 2 == 0) or heads < 1 or k.shape[1] < 1:
        raise ValueError(f"{heads} and {k.shape[1]} heads of {d} channels: heads of an even width up to {MAX_HEAD_DIM} are taken")
    _check_rows("q", q, q)
    _check_rows("k", k, k)
    if k.dtype != q.dtype or k.device != q.device:
        raise ValueError(f"k: {k.dtype} on {k.device}, q is {q.dtype} on {q.device}")
    for name, w in (("wq", wq), ("wk", wk)):
        if w.shape != (d,) or w.dtype not in (torch.bfloat16, torch.float32) or w.dtype != wq.dtype or w.device != q.device \
                or not w.is_contiguous():
            raise ValueError(f"{name}: bf16 or fp32 [{d}] on {q.device}, both alike, got {tuple(w.shape)} {w.dtype} on {w.device}")
    if (cos is None) != (sin is None) or (positions is not None and cos is None):
        raise ValueError("cos and sin come together, positions only with them")
    a = _Args(rows=rows, heads=heads, kv_heads=k.shape[1], d=d, f32=q.dtype == torch.float32, w_bf16=wq.dtype == torch.bfloat16,
              eps=eps, q=_heads(q), k=_heads(k), wq=wq.data_ptr(), wk=wk.data_ptr())
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dim() != 2 or t.shape != cos.shape or t.dtype != torch.float32 or t.device != q.device or not t.is_contiguous():
                raise ValueError(f"{name}: contiguous fp32 [L, rot / 2] on {q.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
        if not 0 <= 2 * cos.shape[1] <= d or (cos.shape[0] < 1 and rows):
            raise ValueError(f"angles {tuple(cos.shape)} for heads of {d} channels")
        a.L, a.rot, a.cos, a.sin = cos.shape[0], 2 * cos.shape[1], cos.data_ptr(), sin.data_ptr()
        if positions is not None:
            if positions.shape != (rows,) or positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device \
                    or not positions.is_contiguous():
                raise ValueError(f"positions: contiguous int32 or int64 [{rows}] on {q.device}, got {tuple(positions.shape)} "
                                 f"{positions.dtype} on {positions.device}")
            a.pos, a.pos64 = positions.data_ptr(), positions.dtype == torch.int64
    for name, t, like in out:
        _check_rows(name, t, like)
        _writable(name, t)
    return a


def qk_norm_fwd(q: torch.Tensor, k: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor, cos: torch.Tensor | None = None,
                sin: torch.Tensor | None = None, *, eps: float, positions: torch.Tensor | None = None,
                q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``q`` [rows, heads, d] and ``k`` [rows, kv_heads, d], bf16 or fp32, with any strides between rows and heads (sections of
    a fused qkv matrix): normed by head with the weights ``wq``, ``wk`` [d] and, with ``cos`` / ``sin``, turned. ``positions``
    [rows] int32 or int64: the table row of every row; one outside the table sets the status word and its row is not written.
    ``q_out``, ``k_out``: where to put the results, memory of their own or ``q`` and ``k`` themselves."""
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else q_out
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device) if k_out is None else k_out
    a = _prepare(q, k, wq, wk, cos, sin, eps, positions, (("q_out", q_out, q), ("k_out", k_out, k)))
    a.q_out, a.k_out = _heads(q_out), _heads(k_out)
    _l.require_cuda(q)
    if a.rows:
        with _l.on_device(q.device):
            a.status = _l.status_word().data_ptr()
            _l.check(_l.lib().aeris_qk_norm_fwd(ctypes.byref(a), _l.stream_ptr()), "aeris_qk_norm_fwd")
    return q_out, k_out


def qk_norm_bwd(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor,
                cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, *, eps: float,
                positions: torch.Tensor | None = None, dq_out: torch.Tensor | None = None, dk_out: torch.Tensor | None = None,
                dwq: torch.Tensor | None = None, dwk: torch.Tensor | None = None):
    """Gradients of :func:`qk_norm_fwd` for ``dq``, ``dk`` with respect to its results; ``q``, ``k`` are its inputs. Returns
    (gradients of q and k, which may overwrite ``dq`` and ``dk``, and fp32 gradients of the weights). ``dwq``, ``dwk`` [d] fp32
    are added to where given. The same bits on every run."""
    dq_out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if dq_out is None else dq_out
    dk_out = torch.empty(k.shape, dtype=k.dtype, device=k.device) if dk_out is None else dk_out
    a = _prepare(q, k, wq, wk, cos, sin, eps, positions, (("dq_out", dq_out, q), ("dk_out", dk_out, k)))
    _check_rows("dq", dq, q)
    _check_rows("dk", dk, k)
    if (dwq is None) != (dwk is None):
        raise ValueError("dwq and dwk come together")
    a.add_dw = dwq is not None
    for name, t in (("dwq", dwq), ("dwk", dwk)):
        if t is not None and (t.shape != wq.shape or t.dtype != torch.float32 or t.device != q.device or not t.is_contiguous()):
            raise ValueError(f"{name}: contiguous fp32 [{a.d}] on {q.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    _l.require_cuda(q)
    if not a.rows:
        return dq_out, dk_out, *(torch.zeros(a.d, dtype=torch.float32, device=q.device) if t is None else t for t in (dwq, dwk))
    if dwq is None:
        dwq, dwk = torch.empty((2, a.d), dtype=torch.float32, device=q.device).unbind(0)
    with _l.on_device(q.device):
        sums = torch.empty((4 * torch.cuda.get_device_properties(q.device).multi_processor_count, 2, a.d), dtype=torch.float32,
                           device=q.device)
        a.dq, a.dk, a.q_out, a.k_out = _heads(dq), _heads(dk), _heads(dq_out), _heads(dk_out)
        a.dwq, a.dwk, a.sums, a.sum_rows = dwq.data_ptr(), dwk.data_ptr(), sums.data_ptr(), sums.shape[0]
        a.status = _l.status_word().data_ptr()
        rc = _l.lib().aeris_qk_norm_bwd(ctypes.byref(a), _l.stream_ptr())
        _l.check(min(rc, 0), "aeris_qk_norm_bwd", kernels=max(rc, 0))
    return dq_out, dk_out, dwq, dwk
