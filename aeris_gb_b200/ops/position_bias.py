"""Python front ends of window attention with a learned bias by relative position (``csrc/position_bias.cu``, ``attention.cu``).

    s[i, j] = scale * q[i] . k[j] + table[bucket(position[i] - position[j]), head]          o = softmax(s) v

Windows of ``high x wide`` tokens in rows. The relative position of query i and key j is the whole number
``(y_i - y_j + high - 1) * (2 * wide - 1) + x_i - x_j + wide - 1``; ``buckets`` maps it to a row of the table. The attention of
:mod:`.attention` is the same without a bias. As all front ends here they record nothing for autograd: the backward pass is a call
of its own.

Scores, softmax statistics and sums are fp32. Probabilities go into the product with v, and into that with dO, in bf16, and so does
the scores' gradient into those with q and k: 2^-8 of every term, for the tensor core multiplies bf16 by bf16 (results 2.0e-3 to
2.5e-3 off where fp32 products end 1.7e-3 off, which is their own rounding). The table's gradient is taken from fp32 values.
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
_TABLES, _INTEGERS = (_F32, _BF16), (torch.int32, torch.int64)


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


def _rows(t, shape, index: int, what: str) -> int:
    """Pitch of rows of bf16. Every attribute is asked for once: they are half of a small call."""
    if t.shape == shape and t.dtype is _BF16 and t.get_device() == index and t.ndim == 2:
        pitch, one = t.stride()
        if one == 1 and (pitch >= shape[1] or shape[0] < 2):
            return pitch if shape[0] > 1 else shape[1]
    raise ValueError(f"{what}: {_BF16} {tuple(shape)} on one device with the others, columns side by side and rows apart, got {_text(t)}")


def _check(qkv, n_win, window, heads, d, table, buckets, scale):
    """Refuses what the kernels cannot take of the inputs that both directions share; returns (high, wide, tokens of a window, pitch
    of qkv, scale, device index)."""
    if len(window) != 2:
        raise ValueError(f"window: (high, wide), got {window!r}")
    high, wide = window
    n, index = high * wide, qkv.get_device()
    if high < 1 or wide < 1 or n > MAX_TOKENS:
        raise ValueError(f"windows of {high} x {wide} tokens: at least one a side, at most {MAX_TOKENS} in all")
    if not (0 <= n_win <= 65535 and 0 < heads <= 65535 and 0 < d <= 128):
        raise ValueError(f"{n_win} windows, {heads} heads of {d} channels: up to 65535, 65535 and 128 are taken")
    pitch = _rows(qkv, (n_win * n, 3 * heads * d), index, "qkv")
    off = (2 * high - 1) * (2 * wide - 1)
    if not (table.ndim == 2 and table.dtype in _TABLES and table.get_device() == index and table.is_contiguous()):
        raise ValueError(f"table: contiguous fp32 or bf16 [rows, {heads}] on {qkv.device}, got {_text(table)}")
    rows, columns = table.shape
    if columns != heads or not 0 < rows * heads < 2 ** 31:
        raise ValueError(f"table: [rows, {heads}], got {_text(table)}")
    if buckets is None:
        if rows != off:
            raise ValueError(f"without buckets the table has a row for each of the {off} relative positions, got {_text(table)}")
    elif not (buckets.shape == (off,) and buckets.dtype in _INTEGERS and buckets.get_device() == index and buckets.is_contiguous()):
        raise ValueError(f"buckets: contiguous int32 or int64 [{off}] on {qkv.device}, got {_text(buckets)}")
    if scale is None:
        scale = d ** -0.5
    elif not math.isfinite(scale):
        raise ValueError(f"scale {scale}")
    return high, wide, n, pitch, scale, index


def _stats(t, shape, index: int, what: str) -> None:
    if not (t.shape == shape and t.dtype is _F32 and t.get_device() == index and t.is_contiguous()):
        raise ValueError(f"{what}: contiguous fp32 {tuple(shape)} on one device with the others, got {_text(t)}")


def _apart(t, others, what: str) -> None:
    for o in others:
        if o is not None and _l.share_memory(t, o):
            raise ValueError(f"{what} lies over another tensor of the call: {_text(t)}, {_text(o)}")


def _launch(name: str, record: bytes, index: int) -> None:
    if torch._C._cuda_getDevice() == index:
        rc = _entry(name)(record, _l.raw_stream())
    else:
        with torch.cuda.device(index):
            rc = _entry(name)(record, _l.raw_stream())
    _l.check(min(rc, 0), name, kernels=max(rc, 0))


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
    high, wide, n, pitch, scale, index = _check(qkv, n_win, window, heads, d, table, buckets, scale)
    tokens, inner = n_win * n, heads * d
    o_pitch = inner
    if out is not None:
        o_pitch = _rows(out, (tokens, inner), index, "out")
        _apart(out, (qkv, table, buckets, lse), "out")
    if lse is not None:
        _stats(lse, (n_win, heads, n), index, "lse")
        _apart(lse, (qkv, table, buckets), "lse")
    _l.require_cuda(qkv)
    if lse is None:
        lse = qkv.new_empty((n_win, heads, n), dtype=_F32)
    # heads and rows of whole 16-byte vectors; others run as zero-padded copies
    tiled = (d | pitch | o_pitch) % 8 == 0 and qkv.data_ptr() % 16 == 0 and (out is None or out.data_ptr() % 16 == 0)
    rows, dp = qkv, d
    if not tiled:
        dp = -(-d // 8) * 8
        rows, pitch, o_pitch = _a._pad_heads(qkv, 3, heads, d, dp), 3 * heads * dp, heads * dp
    o = out if tiled and out is not None else qkv.new_empty((tokens, heads * dp))
    if n_win:
        work, size = 0, _work_bytes(n_win, high, wide, heads, dp, False, False)
        if size:
            buffer = qkv.new_empty(size, dtype=torch.uint8)
            work = buffer.data_ptr()
        _launch("aeris_biased_attn_fwd", _RECORD.pack(
            rows.data_ptr(), o.data_ptr(), lse.data_ptr(), table.data_ptr(), 0 if buckets is None else buckets.data_ptr(), 0, 0, 0, work,
            _l.status_word(qkv.device).data_ptr(), pitch, o_pitch, 0, size, n_win, high, wide, heads, dp, table.shape[0],
            table.dtype is _BF16, buckets is not None and buckets.dtype is torch.int64, 0, scale), index)
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
    put it; ``dtable`` fp32 is added to where given. Rows that hide their pairs get zero. The same bits on every run.

    Probabilities are made anew from ``lse``, in fp32: where all that a query sees has biases of a size B, they are off by about
    1e-7 B of themselves. Entries that are to hide are :data:`HIDDEN` or less.

    Allocates while it runs, in windows of more than 96 tokens, 20 bytes a token and head and, for the table's gradient, sums of
    the scores' gradient of one head (4 bytes a pair of tokens: 4.3 GB in the largest windows) or of more, up to 256 MB."""
    high, wide, n, pitch, scale, index = _check(qkv, n_win, window, heads, d, table, buckets, scale)
    tokens, inner = n_win * n, heads * d
    o_pitch, do_pitch = _rows(o, (tokens, inner), index, "o"), _rows(d_o, (tokens, inner), index, "d_o")
    _stats(lse, (n_win, heads, n), index, "lse")
    g_pitch = 3 * inner
    if dqkv is not None:
        g_pitch = _rows(dqkv, (tokens, 3 * inner), index, "dqkv")
        _apart(dqkv, (qkv, o, d_o, lse, table, buckets, dtable), "dqkv")
    add = dtable is not None
    if add:
        if not need_dtable:
            raise ValueError("a place for a gradient that is not wanted")
        _stats(dtable, table.shape, index, "dtable")
        _apart(dtable, (qkv, o, d_o, lse, table, buckets), "dtable")
    _l.require_cuda(qkv)
    if need_dtable and not add:
        dtable = (qkv.new_empty if n_win else qkv.new_zeros)(table.shape, dtype=_F32)
    tiled = ((d | pitch | o_pitch | do_pitch | g_pitch) % 8 == 0 and qkv.data_ptr() % 16 == 0 and o.data_ptr() % 16 == 0
             and d_o.data_ptr() % 16 == 0 and (dqkv is None or dqkv.data_ptr() % 16 == 0))
    rows, of, do, dp = qkv, o, d_o, d
    if not tiled:
        dp = -(-d // 8) * 8
        rows, of, do = (_a._pad_heads(t, k, heads, d, dp) for t, k in ((qkv, 3), (o, 1), (d_o, 1)))
        pitch, o_pitch, g_pitch = 3 * heads * dp, heads * dp, 3 * heads * dp
    elif o_pitch != do_pitch:
        of, do, o_pitch = o.contiguous(), d_o.contiguous(), inner
    g = dqkv if tiled and dqkv is not None else qkv.new_empty((tokens, 3 * heads * dp))
    if n_win:
        size = _work_bytes(n_win, high, wide, heads, dp, True, need_dtable)
        work = qkv.new_empty(size, dtype=torch.uint8) if size else None
        _launch("aeris_biased_attn_bwd", _RECORD.pack(
            rows.data_ptr(), of.data_ptr(), lse.data_ptr(), table.data_ptr(), 0 if buckets is None else buckets.data_ptr(), do.data_ptr(),
            g.data_ptr(), dtable.data_ptr() if need_dtable else 0, work.data_ptr() if size else 0, _l.status_word(qkv.device).data_ptr(), pitch,
            o_pitch, g_pitch, size, n_win, high, wide, heads, dp, table.shape[0], table.dtype is _BF16,
            buckets is not None and buckets.dtype is torch.int64, add, scale), index)
    if not tiled:
        g = _a._unpad_heads(g, 3, heads, d, dp)
        if dqkv is not None:
            g = dqkv.copy_(g)
    return g, dtable
