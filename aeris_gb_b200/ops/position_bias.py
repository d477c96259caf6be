"""Python front ends of window attention with a learned bias by relative position (``csrc/position_bias.cu``, ``attention.cu``).

    s[i, j] = scale * q[i] . k[j] + table[bucket(position[i] - position[j]), head]          o = softmax(s) v

Windows of ``high x wide`` tokens in rows. The relative position of query i and key j is the whole number
``(y_i - y_j + high - 1) * (2 * wide - 1) + x_i - x_j + wide - 1``; ``buckets`` maps it to a row of the table. The attention of
:mod:`.attention` is the same without a bias.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct

import torch

from . import attention as _a
from . import lib as _l

MAX_TOKENS = 32768          # of a window
HIDDEN = -1e30              # table entries that are no larger hide the pairs of their bucket
# AerisBiasedAttn (csrc/api.h), field by field
_RECORD = struct.Struct("10P4q9if0q")
_BF16, _F32 = torch.bfloat16, torch.float32


def _text(t) -> str:
    return f"{t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}" if isinstance(t, torch.Tensor) else repr(t)


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    f = getattr(_l.lib(), name)
    f.argtypes = (ctypes.c_char_p, ctypes.c_void_p)
    return f


@functools.lru_cache(maxsize=256)
def _work_bytes(n_win: int, high: int, wide: int, heads: int, d: int, backward: bool, with_table: bool) -> int:
    f = _l.lib().aeris_biased_attn_work_bytes
    f.restype = ctypes.c_longlong
    return f(n_win, high, wide, heads, d, int(backward), int(with_table))


def relative_positions(window: tuple[int, int]) -> int:
    """How many relative positions a window of (high, wide) tokens has: entries of ``buckets``, rows of a table without."""
    high, wide = window
    return (2 * high - 1) * (2 * wide - 1)


def _rows(t, shape, dev, what: str, dt=_BF16) -> None:
    if not (t.dim() == 2 and t.shape == shape and t.dtype is dt and t.device == dev and t.stride(1) == 1
            and (shape[0] < 2 or t.stride(0) >= shape[1])):
        raise ValueError(f"{what}: {dt} {tuple(shape)} on {dev} with columns side by side and rows apart, got {_text(t)}")


def _check(qkv, n_win, window, heads, d, table, buckets, scale):
    """Refuses what the kernels cannot take of the inputs that both directions share; returns (high, wide, tokens, scale, device)."""
    if len(window) != 2:
        raise ValueError(f"window: (high, wide), got {window!r}")
    high, wide = window
    n, dev = high * wide, qkv.device
    if high < 1 or wide < 1 or n > MAX_TOKENS:
        raise ValueError(f"windows of {high} x {wide} tokens: at least one a side, at most {MAX_TOKENS} in all")
    if not (0 <= n_win <= 65535 and 0 < heads <= 65535 and 0 < d <= 128):
        raise ValueError(f"{n_win} windows, {heads} heads of {d} channels: up to 65535, 65535 and 128 are taken")
    _rows(qkv, (n_win * n, 3 * heads * d), dev, "qkv")
    off = relative_positions(window)
    if not (table.dim() == 2 and table.shape[1] == heads and table.shape[0] > 0 and table.dtype in (_F32, _BF16)
            and table.device == dev and table.is_contiguous() and table.numel() < 2 ** 31):
        raise ValueError(f"table: contiguous fp32 or bf16 [rows, {heads}] on {dev}, got {_text(table)}")
    if buckets is None:
        if table.shape[0] != off:
            raise ValueError(f"without buckets the table has a row for each of the {off} relative positions, got {_text(table)}")
    elif not (buckets.shape == (off,) and buckets.dtype in (torch.int32, torch.int64) and buckets.device == dev
              and buckets.is_contiguous()):
        raise ValueError(f"buckets: contiguous int32 or int64 [{off}] on {dev}, got {_text(buckets)}")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale {scale}")
    return high, wide, n, scale, dev


def _stats(t, shape, dev, what: str) -> None:
    if not (t.shape == shape and t.dtype is _F32 and t.device == dev and t.is_contiguous()):
        raise ValueError(f"{what}: contiguous fp32 {tuple(shape)} on {dev}, got {_text(t)}")


def _apart(t, others, what: str) -> None:
    for o in others:
        if o is not None and _l.share_memory(t, o):
            raise ValueError(f"{what} lies over another tensor of the call: {_text(t)}, {_text(o)}")


def _record(qkv, o, lse, table, buckets, d_o, dqkv, dtable, work, n_win, high, wide, heads, d, scale, add, dev) -> bytes:
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    pitch = lambda t: 0 if t is None else t.stride(0) if t.shape[0] > 1 else t.shape[1]  # noqa: E731
    return _RECORD.pack(at(qkv), at(o), at(lse), at(table), at(buckets), at(d_o), at(dqkv), at(dtable), at(work),
                        _l.status_word(dev).data_ptr(), pitch(qkv), pitch(o), pitch(dqkv), work.numel(), n_win, high, wide, heads, d,
                        table.shape[0], table.dtype is _BF16, buckets is not None and buckets.dtype is torch.int64, add, scale)


def biased_attn_fwd(qkv: torch.Tensor, n_win: int, window: tuple[int, int], heads: int, d: int, table: torch.Tensor,
                    buckets: torch.Tensor | None = None, *, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                    scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention with a position bias for every (window, head). ``qkv`` is ``[n_win * high * wide, 3 * heads * d]`` bf16 with
    columns ordered (q|k|v, head, channel) and rows window-major, as for :func:`.attention.attn_fwd`; ``d`` up to 128; ``scale``
    is 1 / sqrt(d) where none is given.

    ``table`` [rows, heads] fp32 or bf16; ``buckets`` [relative positions] int32 or int64 names its row for every relative
    position, without them there is a row for each. A bucket outside the table sets the status word. Entries of
    :data:`HIDDEN` and less (-infinity among them) hide the pairs of their bucket; a query that sees nothing gets zeros.

    Returns ``(o [n_win * high * wide, heads * d] bf16, lse [n_win, heads, high * wide] fp32 in the log2 domain, +infinity where a
    query sees nothing)``."""
    high, wide, n, scale, dev = _check(qkv, n_win, window, heads, d, table, buckets, scale)
    if out is not None:
        _rows(out, (n_win * n, heads * d), dev, "out")
        _apart(out, (qkv, table, buckets, lse), "out")
    if lse is not None:
        _stats(lse, (n_win, heads, n), dev, "lse")
        _apart(lse, (qkv, table, buckets), "lse")
    _l.require_cuda(qkv)
    with _l.on_device(dev):
        if lse is None:
            lse = qkv.new_empty((n_win, heads, n), dtype=_F32)
        dp = d if d % 8 == 0 and _a._whole_vectors(qkv) and _a._whole_vectors(out) else -(-d // 8) * 8
        tiled = dp == d and _a._whole_vectors(qkv) and _a._whole_vectors(out)
        rows = qkv if tiled else _a._pad_heads(qkv, 3, heads, d, dp)
        o = out if tiled and out is not None else qkv.new_empty((n_win * n, heads * dp))
        if n_win:
            work = qkv.new_empty(_work_bytes(n_win, high, wide, heads, dp, False, False), dtype=torch.uint8)
            rc = _entry("aeris_biased_attn_fwd")(_record(rows, o, lse, table, buckets, None, None, None, work, n_win, high, wide, heads,
                                                         dp, scale, 0, dev), _l.raw_stream())
            _l.check(min(rc, 0), "aeris_biased_attn_fwd", kernels=max(rc, 0))
        if not tiled:
            o = _a._unpad_heads(o, 1, heads, d, dp)
            if out is not None:
                o = out.copy_(o)
    return o, lse


def biased_attn_bwd(d_o: torch.Tensor, qkv: torch.Tensor, o: torch.Tensor, lse: torch.Tensor, n_win: int, window: tuple[int, int],
                    heads: int, d: int, table: torch.Tensor, buckets: torch.Tensor | None = None, *,
                    dqkv: torch.Tensor | None = None, dtable: torch.Tensor | None = None, need_dtable: bool = True,
                    scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Gradients of :func:`biased_attn_fwd` for ``d_o`` with respect to its first result; ``o``, ``lse`` are its results. Returns
    (gradient of qkv, in its layout; fp32 gradient of the table [rows, heads], or None without ``need_dtable``). ``dqkv``: where to
    put it; ``dtable`` fp32 is added to where given. Rows that hide their pairs get zero. The same bits on every run."""
    high, wide, n, scale, dev = _check(qkv, n_win, window, heads, d, table, buckets, scale)
    _rows(o, (n_win * n, heads * d), dev, "o")
    _rows(d_o, (n_win * n, heads * d), dev, "d_o")
    _stats(lse, (n_win, heads, n), dev, "lse")
    if dqkv is not None:
        _rows(dqkv, tuple(qkv.shape), dev, "dqkv")
        _apart(dqkv, (qkv, o, d_o, lse, table, buckets, dtable), "dqkv")
    if dtable is not None:
        if not need_dtable:
            raise ValueError("a place for a gradient that is not wanted")
        _stats(dtable, tuple(table.shape), dev, "dtable")
        _apart(dtable, (qkv, o, d_o, lse, table, buckets), "dtable")
    _l.require_cuda(qkv)
    with _l.on_device(dev):
        add = dtable is not None
        if need_dtable and dtable is None:
            dtable = (qkv.new_empty if n_win else qkv.new_zeros)(table.shape, dtype=_F32)
        tiled = d % 8 == 0 and all(map(_a._whole_vectors, (qkv, o, d_o, dqkv)))
        dp = -(-d // 8) * 8
        if tiled:
            rows, of, do = qkv, o, d_o
            if of.stride(0) != do.stride(0) and n_win * n > 1:
                of, do = of.contiguous(), do.contiguous()
        else:
            rows, of, do = _a._pad_heads(qkv, 3, heads, d, dp), _a._pad_heads(o, 1, heads, d, dp), _a._pad_heads(d_o, 1, heads, d, dp)
        g = dqkv if tiled and dqkv is not None else qkv.new_empty((n_win * n, 3 * heads * dp))
        if n_win:
            work = qkv.new_empty(_work_bytes(n_win, high, wide, heads, dp, True, need_dtable), dtype=torch.uint8)
            rc = _entry("aeris_biased_attn_bwd")(_record(rows, of, lse, table, buckets, do, g, dtable, work, n_win, high, wide, heads,
                                                         dp, scale, add, dev), _l.raw_stream())
            _l.check(min(rc, 0), "aeris_biased_attn_bwd", kernels=max(rc, 0))
        if not tiled:
            g = _a._unpad_heads(g, 3, heads, d, dp)
            if dqkv is not None:
                g = dqkv.copy_(g)
    return g, dtable
