"""Python front ends of layer norm (``csrc/layer_norm.cu``).

    y = (x - mean) / sqrt(var + eps) * w + b          over the columns of a row

The norm of the plain window transformer block; this framework's own blocks use the modulated RMS norm of
:mod:`.elementwise`. As all front ends here they record nothing for autograd: the backward pass is a call of its own.
"""
from __future__ import annotations

import ctypes
import functools
import struct

import torch

from . import lib as _l

MAX_ROWS = 2 ** 31 - 1
MAX_COLS = 2 ** 31 - 2 ** 10
# AerisLayerNorm (csrc/api.h), field by field
_RECORD = struct.Struct("10P4q5if0q")
_FLOATS = (torch.bfloat16, torch.float32)


def _text(t) -> str:
    return f"{t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}" if isinstance(t, torch.Tensor) else repr(t)


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    f = getattr(_l.lib(), name)
    f.argtypes = (ctypes.c_char_p, ctypes.c_void_p)
    return f


@functools.lru_cache(maxsize=None)
def _multiprocessors(device: int) -> int:
    return torch.cuda.get_device_properties(device).multi_processor_count


def _launch(name: str, record: bytes, index: int) -> None:
    if torch._C._cuda_getDevice() == index:
        rc = _entry(name)(record, _l.raw_stream())
    else:
        with torch.cuda.device(index):
            rc = _entry(name)(record, _l.raw_stream())
    _l.check(min(rc, 0), name, kernels=max(rc, 0))


def _vector(t, cols: int, index: int) -> bool:
    return t.shape == (cols,) and t.dtype in _FLOATS and t.get_device() == index and t.is_contiguous()


def _check(x, w, b):
    """Refuses what the kernels cannot take of the inputs that both directions share; returns (rows, cols, pitch, type, device index).
    Every attribute is asked for once: they are half of a small call."""
    dt, index = x.dtype, x.get_device()
    if x.ndim != 2 or dt not in _FLOATS:
        raise ValueError(f"x [rows, cols] in bf16 or fp32, got {_text(x)}")
    rows, cols = x.shape
    if rows > MAX_ROWS or not 0 < cols <= MAX_COLS:
        raise ValueError(f"{rows} rows of {cols} columns: at most {MAX_ROWS} of 1 to {MAX_COLS} are taken")
    pitch, one = x.stride()
    if one != 1 and cols > 1:
        raise ValueError(f"columns lie side by side, got {_text(x)}")
    if w is not None and not _vector(w, cols, index) or b is not None and not _vector(b, cols, index):
        raise ValueError(f"weight and bias: contiguous bf16 or fp32 [{cols}] on {x.device}, got {_text(w)} and {_text(b)}")
    if w is not None and b is not None and w.dtype is not b.dtype:
        raise ValueError(f"weight and bias are of one type, got {w.dtype} and {b.dtype}")
    return rows, cols, pitch, dt, index


def _like(t, shape, dt, index, what: str) -> int:
    """Pitch of a second matrix of the same form."""
    if t.shape == shape and t.dtype is dt and t.get_device() == index:
        pitch, one = t.stride()
        if one == 1 or shape[1] == 1:
            return pitch
    raise ValueError(f"{what}: {dt} {tuple(shape)} on the device of x with columns side by side, got {_text(t)}")


def _result(t, shape, dt, index, what: str, *inputs) -> int:
    """Pitch of a matrix that is written: rows apart, and in the place of an input only element by element."""
    pitch = _like(t, shape, dt, index, what)
    if shape[0] > 1 and pitch < shape[1]:
        raise ValueError(f"{what}: rows lie over one another, got {_text(t)}")
    for i in inputs:
        if i is not None and i is not t and _l.share_memory(t, i) and not (i.shape == shape and _l.same_memory(t, i)):
            raise ValueError(f"{what} lies beside an input's elements: {_text(t)}, {_text(i)}")
    return pitch


def layer_norm_fwd(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *, eps: float,
                   out: torch.Tensor | None = None, stats: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``x`` [rows, cols] bf16 or fp32, rows of any pitch (a section of a wider matrix). Returns (normed rows in x's type, fp32
    [rows, 2]: mean and 1 / sqrt(var + eps) of every row, which :func:`layer_norm_bwd` takes; from an 8-byte boundary on). ``weight``, ``bias`` [cols] bf16 or
    fp32, each may be missing. ``out`` may be ``x`` itself."""
    rows, cols, pitch, dt, index = _check(x, weight, bias)
    if out is not None:
        pitch_out = _result(out, x.shape, dt, index, "out", x, weight, bias)
    if stats is not None:
        if not _stats(stats, rows, index):
            raise ValueError(f"stats: contiguous fp32 [{rows}, 2] from an 8-byte boundary on, on {x.device}, got {_text(stats)}")
        if any(t is not None and _l.share_memory(stats, t) for t in (x, weight, bias, out)):
            raise ValueError("stats lie over another tensor of the call")
    _l.require_cuda(x)
    if out is None:
        out, pitch_out = (torch.empty_like(x) if pitch == cols else x.new_empty((rows, cols))), cols
    if stats is None:
        stats = x.new_empty((rows, 2), dtype=torch.float32)
    if rows:
        w_f32 = (weight if weight is not None else bias if bias is not None else x).dtype is torch.float32
        _launch("aeris_layer_norm_fwd", _RECORD.pack(
            x.data_ptr(), 0, out.data_ptr(), 0 if weight is None else weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
            stats.data_ptr(), 0, 0, 0, _l.status_word(x.device).data_ptr(), rows, pitch, 0, max(pitch_out, cols), cols, dt is torch.float32, w_f32, 0, 0, eps), index)
    return out, stats


def _stats(t, rows: int, index: int) -> bool:
    """Mean and reciprocal deviation of a row are read and written as one: from an 8-byte boundary on."""
    return (t.shape == (rows, 2) and t.dtype is torch.float32 and t.get_device() == index and t.is_contiguous()
            and t.data_ptr() % 8 == 0)


def layer_norm_bwd(dy: torch.Tensor, x: torch.Tensor, stats: torch.Tensor, weight: torch.Tensor | None = None, *,
                   bias: bool = True, dx: torch.Tensor | None = None, dw: torch.Tensor | None = None,
                   db: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """Gradients of :func:`layer_norm_fwd` for ``dy`` with respect to its rows; ``x`` and ``stats`` are its input and its second
    result. Returns (gradient of x in x's type, fp32 gradient of the weight or None without one, fp32 gradient of the bias or None
    with ``bias=False``). ``dx`` may be ``dy`` or ``x`` itself; ``dw``, ``db`` [cols] fp32 are added to where given. The same
    bits on every run; tensors whose rows start elsewhere may be added up in another order. Allocates :func:`slices_for` times 8
    bytes a column for the sums while it runs."""
    rows, cols, pitch, dt, index = _check(x, weight, None)
    shape = x.shape
    pitch_dy = _like(dy, shape, dt, index, "dy")
    if not _stats(stats, rows, index):
        raise ValueError(f"stats: contiguous fp32 [{rows}, 2] from an 8-byte boundary on, on {x.device}, got {_text(stats)}")
    add = dw is not None or db is not None
    if add:
        if weight is None and dw is not None or not bias and db is not None:
            raise ValueError("a gradient to add to without the parameter")
        if (weight is not None) != (dw is not None) or bias != (db is not None):
            raise ValueError("dw and db come together")
        for t in (dw, db):
            if t is not None and not (_vector(t, cols, index) and t.dtype is torch.float32):
                raise ValueError(f"dw and db: contiguous fp32 [{cols}] on {x.device}, got {_text(t)}")
        if dw is not None and db is not None and _l.share_memory(dw, db):
            raise ValueError("dw and db are in the same memory")
        if any(_l.share_memory(t, u) for t in (dw, db) if t is not None for u in (dy, x, stats, weight) if u is not None):
            raise ValueError("dw or db lies over an input")
    if dx is not None:
        pitch_dx = _result(dx, shape, dt, index, "dx", dy, x)
        if any(t is not None and _l.share_memory(dx, t) for t in (stats, weight, dw, db)):
            raise ValueError("dx lies over another tensor of the call")
    _l.require_cuda(x)
    if dx is None:
        dx, pitch_dx = (torch.empty_like(x) if pitch == cols else x.new_empty((rows, cols))), cols
    if not add:
        make = x.new_empty if rows else x.new_zeros
        if weight is not None:
            dw = make((cols,), dtype=torch.float32)
        if bias:
            db = make((cols,), dtype=torch.float32)
    if rows:
        slices, work = 0, None
        if dw is not None or db is not None:
            slices = slices_for(rows, cols, _multiprocessors(index))
            if slices > 1:
                work = x.new_empty((slices, 2, cols), dtype=torch.float32)
        _launch("aeris_layer_norm_bwd", _RECORD.pack(
            x.data_ptr(), dy.data_ptr(), dx.data_ptr(), 0 if weight is None else weight.data_ptr(), 0, stats.data_ptr(),
            0 if dw is None else dw.data_ptr(), 0 if db is None else db.data_ptr(), 0 if work is None else work.data_ptr(),
            _l.status_word(x.device).data_ptr(), rows, pitch, pitch_dy, max(pitch_dx, cols), cols, dt is torch.float32, weight is not None and weight.dtype is torch.float32,
            add, slices, 0.0), index)
    return dx, dw, db


def slices_for(rows: int, cols: int, multiprocessors: int) -> int:
    """Slices of the rows whose column sums may be taken apart: four blocks on every multiprocessor, four rows each; one block and
    one row where rows are wide, for a slice is as large as two of them (2,000 x 65,536 bf16: 868 us a call and 74 MB of sums, with four
    blocks 1,489 and 296; 4,000 x 5,000 51 us and 6 MB, 51 and 23). One slice for what a cluster of blocks, which joins its own
    sums, is through with before a second launch would begin (221 x 35, bf16: 15.7 us a call for 20.1; 250 x 200: 14.0 for 18.9, in a
    graph 9.4 for 9.6)."""
    if rows <= 256 and rows * cols <= 2 ** 16 and cols <= 4096:
        return 1
    return max(2, min(4 * multiprocessors, -(-rows // 4)) if cols <= 4096 else min(multiprocessors, rows))
