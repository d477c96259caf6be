"""Python front ends of the norms of queries and keys by head with the position rotation (``csrc/qk_norm.cu``).

    z = w * x / sqrt(mean(x^2) + eps)          over the channels of one head, ``w`` shared by the heads
    y[2i], y[2i + 1] = z turned by the angle of (position, i)

The convention of :func:`.elementwise.rope_qk_`: neighbouring channels form a pair, ``cos`` / ``sin`` [L, rot / 2] fp32 hold the
angles of every position, row r of a window-major stream is at position r mod L unless ``positions`` says otherwise.
"""
from __future__ import annotations

import ctypes
import functools
import struct

import torch

from . import lib as _l

MAX_HEAD_DIM = 256
MAX_ROWS = 2 ** 31 - 2 ** 21
# AerisQkNorm (csrc/api.h), field by field: packing 39 values takes 0.4 us, filling a ctypes.Structure with them 12.
_RECORD = struct.Struct("Pqq" * 6 + "9P" + "q" + "10i" + "f" + "0q")
_FLOATS = (torch.bfloat16, torch.float32)
_INTEGERS = (torch.int32, torch.int64)


def _like(t: torch.Tensor, shape, dtype, device) -> bool:
    return t.shape == shape and t.dtype is dtype and t.device == device and (t.is_contiguous() or t.stride(2) == 1)


def _apart(t: torch.Tensor) -> bool:
    """Whether no two elements of ``t`` share an address (expanded rows or heads would be written by several warps)."""
    (rows, heads, d), (row, head, _) = t.shape, t.stride()
    return (((heads == 1 or head >= d) and (rows == 1 or row >= (heads - 1) * head + d))
            or ((rows == 1 or row >= d) and (heads == 1 or head >= (rows - 1) * row + d)) or t.numel() == 0)


def _text(t) -> str:
    return f"{t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}" if isinstance(t, torch.Tensor) else repr(t)


def _check_more(shape, dt, dev, *tensors) -> None:
    for t in tensors:
        if t is not None and not _like(t, shape, dt, dev):
            raise ValueError(f"{dt} {tuple(shape)} on {dev} with channels side by side, got {_text(t)}")


def _share(a: tuple, b: tuple, rows: int, d: int, size: int) -> bool:
    """:func:`.lib.share_memory` of (tensor [rows, heads, d], address, row pitch, head pitch, heads), without asking tensors again
    where ranges of memory lie apart or rows are one piece each."""
    t, at, row, head, heads = a
    u, to, pitch, u_head, u_heads = b
    if at >= to + ((rows - 1) * pitch + (u_heads - 1) * u_head + d) * size or to >= at + ((rows - 1) * row + (heads - 1) * head + d) * size:
        return False
    if row != pitch or row <= 0 or (head != d and heads > 1) or (u_head != d and u_heads > 1):
        return _l.share_memory(t, u)
    off, row = at - to, row * size
    m = max((-heads * d * size - off) // row + 1, 1 - rows)
    return m < rows and off + m * row < u_heads * d * size


def _check_results(q_out, k_out, of_q: tuple, of_k: tuple, rows: int, d: int) -> None:
    """``of_q``, ``of_k``: inputs of q's and k's kernels. Either result may take the place of one of its own. One that lies over
    the other's, or beside an input's elements, would be written while other warps read there."""
    for t in (q_out, k_out):
        if t is not None and not t.is_contiguous() and not _apart(t):
            raise ValueError(f"elements of a result share addresses: {_text(t)}")
    if not rows:
        return
    size = of_q[0].element_size()
    places = [[(t, t.data_ptr(), *t.stride()[:2], heads) for t in ts if t is not None]
              for heads, ts in ((of_q[0].shape[1], (q_out, *of_q)), (of_k[0].shape[1], (k_out, *of_k)))]
    for t, mine, others in ((q_out, *places), (k_out, *places[::-1])):
        if t is None:
            continue
        for b in others[-len(of_q):]:
            if _share(mine[0], b, rows, d, size):
                raise ValueError(f"a result of q lies over k or one of k over q: {_text(t)}, {_text(b[0])}")
        for b in mine[1:]:
            if t is not b[0] and _share(mine[0], b, rows, d, size) and not _l.same_memory(t, b[0]):
                raise ValueError(f"a result lies beside its input's elements: {_text(t)}, {_text(b[0])}")
    if q_out is not None and k_out is not None and _share(places[0][0], places[1][0], rows, d, size):
        raise ValueError("the results of q and k are in the same memory")


def _check_dw(dwq, dwk, d: int, dev) -> None:
    for t in (dwq, dwk):
        if t.shape != (d,) or t.dtype is not torch.float32 or t.device != dev or not t.is_contiguous():
            raise ValueError(f"gradients of the weights: contiguous fp32 [{d}] on {dev}, got {_text(t)}")
    if 0 < abs(dwq.data_ptr() - dwk.data_ptr()) < 4 * d:
        raise ValueError("gradients of the weights that overlap are the same tensor, a weight's that q and k share")


def _check(q, k, wq, wk, cos, sin, positions):
    """Refuses what the kernels cannot take of the inputs that both directions share; returns (shape of q, of k, strides of q,
    of k, type, device, table length, rotated channels). Every attribute is asked for once: they are half of a small call."""
    qs, ks, dt, dev = q.shape, k.shape, q.dtype, q.device
    if len(qs) != 3 or len(ks) != 3 or qs[0] != ks[0] or qs[2] != ks[2] or dt not in _FLOATS:
        raise ValueError(f"q [rows, heads, d] and k [rows, kv_heads, d] in bf16 or fp32, got {_text(q)} and {_text(k)}")
    rows, heads, d = qs
    if rows > MAX_ROWS:
        raise ValueError(f"{rows} rows: at most {MAX_ROWS} are taken")
    if not 0 < d <= MAX_HEAD_DIM or d % 2 or heads < 1 or ks[1] < 1:
        raise ValueError(f"{heads} and {ks[1]} heads of {d} channels: heads of an even width up to {MAX_HEAD_DIM} are taken")
    q_at, k_at = q.stride(), k.stride()
    if not (q_at[2] == 1 == k_at[2]) or k.dtype is not dt or k.device != dev:
        raise ValueError(f"q and k: one type, one device, channels side by side, got {_text(q)} and {_text(k)}")
    w_dt, one = wq.dtype, (d,)
    if not (wq.shape == one == wk.shape and w_dt in _FLOATS and w_dt is wk.dtype and wq.device == dev == wk.device
            and wq.is_contiguous() and wk.is_contiguous()):
        raise ValueError(f"weights: bf16 or fp32 [{d}] on {dev}, both alike, got {_text(wq)} and {_text(wk)}")
    if cos is None or sin is None:
        if cos is not None or sin is not None or positions is not None:
            raise ValueError("cos and sin come together, positions only with them")
        return qs, ks, q_at, k_at, dt, dev, 0, 0
    table = cos.shape
    if not (len(table) == 2 and sin.shape == table and cos.dtype is torch.float32 is sin.dtype and cos.device == dev == sin.device
            and cos.is_contiguous() and sin.is_contiguous() and 2 * table[1] <= d and (table[0] > 0 or not rows)):
        raise ValueError(f"angles: contiguous fp32 [L, at most {d // 2}] on {dev}, got {_text(cos)} and {_text(sin)}")
    if positions is not None and not (positions.shape == (rows,) and positions.dtype in _INTEGERS
                                      and positions.device == dev and positions.is_contiguous()):
        raise ValueError(f"positions: contiguous int32 or int64 [{rows}] on {dev}, got {_text(positions)}")
    return qs, ks, q_at, k_at, dt, dev, table[0], 2 * table[1]


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    f = getattr(_l.lib(), name)
    f.argtypes = (ctypes.c_char_p, ctypes.c_void_p)
    return f


@functools.lru_cache(maxsize=None)
def _multiprocessors(device: int) -> int:
    return torch.cuda.get_device_properties(device).multi_processor_count


def _launch(name: str, record: bytes, dev) -> int:
    if torch._C._cuda_getDevice() == dev.index:
        return _entry(name)(record, _l.raw_stream())
    with torch.cuda.device(dev):
        return _entry(name)(record, _l.raw_stream())


def qk_norm_fwd(q: torch.Tensor, k: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor, cos: torch.Tensor | None = None,
                sin: torch.Tensor | None = None, *, eps: float, positions: torch.Tensor | None = None,
                q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``q`` [rows, heads, d] and ``k`` [rows, kv_heads, d], bf16 or fp32, with any strides between rows and heads (sections of
    a fused qkv matrix): normed by head with the weights ``wq``, ``wk`` [d] and, with ``cos`` / ``sin``, turned. ``positions``
    [rows] int32 or int64: the table row of every row; one outside the table sets the status word and its row is not written.
    ``q_out``, ``k_out``: where to put the results, memory of their own or ``q`` and ``k`` themselves; results that lie over
    anything else of them are refused."""
    qs, ks, q_at, k_at, dt, dev, length, rot = _check(q, k, wq, wk, cos, sin, positions)
    rows, heads, d = qs
    if q_out is not None or k_out is not None:
        _check_more(qs, dt, dev, q_out)
        _check_more(ks, dt, dev, k_out)
        _check_results(q_out, k_out, (q,), (k,), rows, d)
    _l.require_cuda(q)
    q_row, q_head, k_row, k_head = heads * d, d, ks[1] * d, d
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        q_row, q_head, _ = q_out.stride()
    if k_out is None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    else:
        k_row, k_head, _ = k_out.stride()
    if rows:
        record = _RECORD.pack(q.data_ptr(), q_at[0], q_at[1], k.data_ptr(), k_at[0], k_at[1], 0, 0, 0, 0, 0, 0, q_out.data_ptr(),
                              q_row, q_head, k_out.data_ptr(), k_row, k_head, wq.data_ptr(), wk.data_ptr(),
                              cos.data_ptr() if rot else 0, sin.data_ptr() if rot else 0,
                              0 if positions is None else positions.data_ptr(), 0, 0, 0, _l.status_word(dev).data_ptr(), rows, length,
                              heads, ks[1], d, rot, dt is torch.float32, wq.dtype is torch.bfloat16,
                              positions is not None and positions.dtype is torch.int64, 0, 0, eps)
        _l.check(_launch("aeris_qk_norm_fwd", record, dev), "aeris_qk_norm_fwd")
    return q_out, k_out


def qk_norm_bwd(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor,
                cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, *, eps: float,
                positions: torch.Tensor | None = None, dq_out: torch.Tensor | None = None, dk_out: torch.Tensor | None = None,
                dwq: torch.Tensor | None = None, dwk: torch.Tensor | None = None):
    """Gradients of :func:`qk_norm_fwd` for ``dq``, ``dk`` with respect to its results; ``q``, ``k`` are its inputs. Returns
    (gradients of q and k, which may overwrite ``dq`` and ``dk`` element by element, and fp32 gradients of the weights). ``dwq``,
    ``dwk`` [d] fp32 are added to where given, and may be one tensor, of a weight that q and k share. A row whose position lies
    outside the table adds nothing, and its gradients are not written. The same bits on every run."""
    add = dwq is not None
    if add != (dwk is not None):
        raise ValueError("dwq and dwk come together")
    qs, ks, q_at, k_at, dt, dev, length, rot = _check(q, k, wq, wk, cos, sin, positions)
    rows, heads, d = qs
    _check_more(qs, dt, dev, dq, dq_out)
    _check_more(ks, dt, dev, dk, dk_out)
    if dq_out is not None or dk_out is not None:
        _check_results(dq_out, dk_out, (dq, q), (dk, k), rows, d)
    if add:
        _check_dw(dwq, dwk, d, dev)
    _l.require_cuda(q)
    q_row, q_head, k_row, k_head = heads * d, d, ks[1] * d, d
    if dq_out is None:
        dq_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        q_row, q_head, _ = dq_out.stride()
    if dk_out is None:
        dk_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    else:
        k_row, k_head, _ = dk_out.stride()
    if not add:
        make = torch.empty_like if rows else torch.zeros_like
        dwq, dwk = make(wq, dtype=torch.float32), make(wk, dtype=torch.float32)
    if rows:
        blocks = 4 * _multiprocessors(dev.index)
        sums = q.new_empty((blocks, d), dtype=torch.float32)
        dq_row, dq_head, _ = dq.stride()
        dk_row, dk_head, _ = dk.stride()
        record = _RECORD.pack(q.data_ptr(), q_at[0], q_at[1], k.data_ptr(), k_at[0], k_at[1], dq.data_ptr(), dq_row, dq_head,
                              dk.data_ptr(), dk_row, dk_head, dq_out.data_ptr(), q_row, q_head, dk_out.data_ptr(), k_row, k_head,
                              wq.data_ptr(), wk.data_ptr(), cos.data_ptr() if rot else 0, sin.data_ptr() if rot else 0,
                              0 if positions is None else positions.data_ptr(), dwq.data_ptr(), dwk.data_ptr(), sums.data_ptr(),
                              _l.status_word(dev).data_ptr(), rows, length, heads, ks[1], d, rot, dt is torch.float32,
                              wq.dtype is torch.bfloat16, positions is not None and positions.dtype is torch.int64, add, blocks, eps)
        rc = _launch("aeris_qk_norm_bwd", record, dev)
        _l.check(min(rc, 0), "aeris_qk_norm_bwd", kernels=max(rc, 0))
    return dq_out, dk_out, dwq, dwk
