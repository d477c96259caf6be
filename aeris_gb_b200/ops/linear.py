"""Python front ends of linear layers with bias, activation and residual in one product (``csrc/linear.cu``).

    z = x @ w^T + b          y = resid + act(z)

The layers of the plain window transformer block; this framework's own blocks use the products of :mod:`.gemm`, without biases
and with gates. As all front ends here they record nothing for autograd: the backward pass is a call of its own.
"""
from __future__ import annotations

import ctypes
import functools
import struct

import torch

from . import lib as _l

ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")
_ACT = {name: i for i, name in enumerate(ACTIVATIONS)}
MOST = 2 ** 31 - 2 ** 12         # rows, columns
# AerisLinear, AerisLinearGrad (csrc/api.h), field by field
_FORWARD = struct.Struct("8P6q5i0q")
_GRAD = struct.Struct("9P7q6i0q")
_BF16, _F32 = torch.bfloat16, torch.float32
_BIAS = (_F32, _BF16)


def _text(t) -> str:
    return f"{t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}" if isinstance(t, torch.Tensor) else repr(t)


@functools.lru_cache(maxsize=None)
def _entry(name: str, sizes: int = 0):
    f = getattr(_l.lib(), name)
    f.argtypes = (ctypes.c_int,) * sizes or (ctypes.c_char_p, ctypes.c_void_p)
    f.restype = ctypes.c_longlong if sizes else ctypes.c_int
    return f


@functools.lru_cache(maxsize=1024)
def _bytes(name: str, *sizes: int) -> int:
    return _entry(name, len(sizes))(*sizes)


def _launch(name: str, record: bytes, index: int) -> None:
    if torch._C._cuda_getDevice() == index:
        rc = _entry(name)(record, _l.raw_stream())
    else:
        with torch.cuda.device(index):
            rc = _entry(name)(record, _l.raw_stream())
    _l.check(min(rc, 0), name, kernels=max(rc, 0))


def _matrix(t, shape, index: int, what: str, dtype=_BF16) -> int:
    """Pitch of a matrix of the given shape. Every attribute is asked for once: they are half of a small call."""
    if t.shape == shape and t.dtype is dtype and t.get_device() == index and t.ndim == 2:
        pitch, one = t.stride()
        if one == 1 or shape[1] == 1:
            return pitch
    raise ValueError(f"{what}: {dtype} {tuple(shape)} on one device with the others, columns side by side, got {_text(t)}")


def _result(t, shape, index: int, what: str, *others, dtype=_BF16, inside=None) -> int:
    """``inside``: the one input that the result may take the place of, element by element (where it is none of ``others``, too)."""
    pitch = _matrix(t, shape, index, what, dtype)
    if shape[0] > 1 and pitch < shape[1]:
        raise ValueError(f"{what}: rows lie over one another, got {_text(t)}")
    if inside is not None and not _l.same_memory(t, inside):
        others += inside,
    for o in others:
        if o is not None and _l.share_memory(t, o):
            raise ValueError(f"{what} lies over another tensor of the call: {_text(t)}, {_text(o)}")
    return pitch


def _check(x, w):
    """(rows, inner, columns, pitches of x and w, device index)"""
    if x.ndim != 2 or w.ndim != 2 or x.dtype is not _BF16:
        raise ValueError(f"x [rows, inner] and w [cols, inner] in bf16, got {_text(x)} and {_text(w)}")
    shape, other, index = x.shape, w.shape, x.get_device()
    rows, inner = shape
    cols, _ = other
    if not (rows <= MOST and 0 < inner <= MOST and 0 < cols <= MOST):
        raise ValueError(f"x {tuple(shape)}, w {tuple(other)}: 1 to {MOST} of each (rows: none, too)")
    return rows, inner, cols, _matrix(x, shape, index, "x"), _matrix(w, (cols, inner), index, "w"), index


def _act_code(act: str) -> int:
    code = _ACT.get(act)
    if code is None:
        raise ValueError(f"act is one of {', '.join(ACTIVATIONS)}, got {act!r}")
    return code


def _padded(at: int, rows: int, cols: int, pitch: int) -> bool:
    """Whether a product takes a copy of a matrix whose rows start on 16-byte boundaries, as tiled loads need it."""
    return at % 16 != 0 or (rows > 1 and (pitch % 8 != 0 or pitch < cols))


def linear_fwd(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, *, act: str = "none",
               resid: torch.Tensor | None = None, keep: bool = False, out: torch.Tensor | None = None,
               z: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``resid + act(x @ w^T + bias)`` for ``x`` [rows, inner] and ``w`` [cols, inner], bf16; ``bias`` [cols] fp32 or bf16 and
    ``resid`` [rows, cols] bf16 may be missing. ``act``: one of :data:`ACTIVATIONS` ("gelu" by the error function, absolutely 2.1e-7
    off at most, relatively more than a rounding to bf16 where it is below 6e-9; "gelu_tanh" by the hyperbolic tangent). Returns (the result, and with ``keep`` the values before the activation, bias included, which
    :func:`linear_bwd` takes: else None). ``out``, ``z``: where to put them; ``out`` may be ``resid`` itself, where that is neither ``x`` nor ``w``.

    Any sizes and pitches. Rows that start on 16-byte boundaries are fastest: others of ``x`` and ``w`` are copied first, others of
    the results, and those of columns that are no multiple of 8, are written element by element."""
    rows, inner, cols, x_pitch, w_pitch, index = _check(x, w)
    code = _act_code(act)
    shape = (rows, cols)
    if bias is not None and not (bias.shape == (cols,) and bias.dtype in _BIAS and bias.get_device() == index and bias.is_contiguous()):
        raise ValueError(f"bias: contiguous fp32 or bf16 [{cols}] on {x.device}, got {_text(bias)}")
    r_pitch = 0 if resid is None else _matrix(resid, shape, index, "resid")
    if z is not None and not keep:
        raise ValueError("z is written with keep=True")
    y_pitch = z_pitch = cols
    if out is not None:
        y_pitch = _result(out, shape, index, "out", x, w, bias, z, inside=resid)
    if z is not None:
        z_pitch = _result(z, shape, index, "z", x, w, bias, resid)
    _l.require_cuda(x)
    if out is None:
        out = x.new_empty(shape)
    if keep and z is None:
        z = x.new_empty(shape)
    if rows:
        at, w_at, work, n = x.data_ptr(), w.data_ptr(), 0, 0
        pad = _padded(at, rows, inner, x_pitch), _padded(w_at, cols, inner, w_pitch)
        if pad[0] or pad[1]:
            n = _bytes("aeris_linear_fwd_bytes", rows, inner, cols, *pad)
            buffer = x.new_empty(n, dtype=torch.uint8)
            work = buffer.data_ptr()
        _launch("aeris_linear_fwd", _FORWARD.pack(
            at, w_at, 0 if bias is None else bias.data_ptr(), 0 if resid is None else resid.data_ptr(), out.data_ptr(),
            z.data_ptr() if keep else 0, work, _l.status_word(x.device).data_ptr(), x_pitch, w_pitch, r_pitch, y_pitch, z_pitch, n,
            rows, inner, cols, code, bias is not None and bias.dtype is _BF16), index)
    return out, z


def linear_bwd(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, z: torch.Tensor | None = None, *, act: str = "none",
               bias: bool = True, need_dx: bool = True, need_dw: bool = True, dx: torch.Tensor | None = None,
               dw: torch.Tensor | None = None, db: torch.Tensor | None = None):
    """Gradients of :func:`linear_fwd` for ``dy`` [rows, cols] bf16; ``z`` is its second result (not asked for with act="none").
    Returns (gradient of x in bf16 or None, of w in bf16 or None, of the bias in fp32 or, with ``bias=False``, None). The
    gradient of ``resid`` is ``dy``. ``dx``: where to put that of x, not over any input. ``dw`` [cols, inner] and ``db`` [cols], both
    fp32, are added to where given. The same bits on every run.

    The gradient of z is rounded to bf16 for both products (2^-8 of every term); ``db`` sums it before."""
    rows, inner, cols, x_pitch, w_pitch, index = _check(x, w)
    code = _act_code(act)
    shape = (rows, cols)
    dy_pitch = _matrix(dy, shape, index, "dy")
    z_pitch = 0
    if code:
        if z is None:
            raise ValueError(f"act={act!r}: the backward pass takes z, the values before the activation")
        z_pitch = _matrix(z, shape, index, "z")
    else:
        z = None
    dx_pitch = dw_pitch = inner
    add_db, dw_f32 = db is not None, dw is not None
    if dx is not None:
        if not need_dx:
            raise ValueError("a place for a gradient that is not wanted")
        dx_pitch = _result(dx, (rows, inner), index, "dx", dy, x, w, z, dw, db)
    if dw_f32:
        if not need_dw:
            raise ValueError("a place for a gradient that is not wanted")
        dw_pitch = _result(dw, (cols, inner), index, "dw", dy, x, w, z, db, dtype=_F32)
    if add_db:
        if not bias:
            raise ValueError("a place for a gradient that is not wanted")
        if not (db.shape == (cols,) and db.dtype is _F32 and db.get_device() == index and db.is_contiguous()):
            raise ValueError(f"db: contiguous fp32 [{cols}] on {x.device}, got {_text(db)}")
        if any(t is not None and _l.share_memory(db, t) for t in (dy, x, w, z)):
            raise ValueError("db lies over an input")
    _l.require_cuda(x)
    make = x.new_empty if rows else x.new_zeros
    if need_dx and dx is None:
        dx = make((rows, inner))
    if need_dw and dw is None:
        dw = make((cols, inner))
    if bias and db is None:
        db = make((cols,), dtype=_F32)
    if rows and (need_dx or need_dw or bias):
        dy_at, x_at, w_at, work = dy.data_ptr(), x.data_ptr(), w.data_ptr(), 0
        n = _bytes("aeris_linear_bwd_bytes", rows, inner, cols, code != 0 or _padded(dy_at, rows, cols, dy_pitch),
                   _padded(x_at, rows, inner, x_pitch), _padded(w_at, cols, inner, w_pitch), need_dx, need_dw, bias, dw_f32)
        if n:
            buffer = x.new_empty(n, dtype=torch.uint8)
            work = buffer.data_ptr()
        _launch("aeris_linear_bwd", _GRAD.pack(
            dy_at, x_at, w_at, 0 if z is None else z.data_ptr(), dx.data_ptr() if need_dx else 0, dw.data_ptr() if need_dw else 0,
            db.data_ptr() if bias else 0, work, _l.status_word(x.device).data_ptr(), dy_pitch, x_pitch, w_pitch, z_pitch, dx_pitch,
            dw_pitch, n, rows, inner, cols, code, dw_f32, add_db), index)
    return dx, dw, db
