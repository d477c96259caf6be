"""Python front ends of linear layers with bias, activation and residual in one product (``csrc/linear.cu``).

    z = x @ w^T + b          y = resid + act(z)

The layers of the plain window transformer block; this framework's own blocks use the products of :mod:`.gemm`, without biases
and with gates.
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


def _launch(name: str, record: bytes, dev) -> None:
    if torch._C._cuda_getDevice() == dev.index:
        rc = _entry(name)(record, _l.raw_stream())
    else:
        with torch.cuda.device(dev):
            rc = _entry(name)(record, _l.raw_stream())
    _l.check(min(rc, 0), name, kernels=max(rc, 0))


def _matrix(t, shape, dev, what: str, dtypes=(_BF16,)) -> None:
    if not (t.dim() == 2 and t.shape == shape and t.dtype in dtypes and t.device == dev):
        raise ValueError(f"{what}: {dtypes[0]} {tuple(shape)} on {dev}, got {_text(t)}")
    if (t.stride(1) != 1 and shape[1] > 1) or t.stride(0) < 0:
        raise ValueError(f"{what}: columns lie side by side, got {_text(t)}")


def _result(t, shape, dev, what: str, *others, dtypes=(_BF16,), inside=None) -> None:
    """``inside``: the one input that the result may take the place of, element by element."""
    _matrix(t, shape, dev, what, dtypes)
    if shape[0] > 1 and t.stride(0) < shape[1]:
        raise ValueError(f"{what}: rows lie over one another, got {_text(t)}")
    for o in others:
        if o is not None and _l.share_memory(t, o) and not (o is inside and _l.same_memory(t, o)):
            raise ValueError(f"{what} lies over another tensor of the call: {_text(t)}, {_text(o)}")


def _check(x, w):
    if x.dim() != 2 or w.dim() != 2 or x.dtype is not _BF16:
        raise ValueError(f"x [rows, inner] and w [cols, inner] in bf16, got {_text(x)} and {_text(w)}")
    (rows, inner), cols, dev = x.shape, w.shape[0], x.device
    if max(rows, inner, cols) > MOST or inner < 1 or cols < 1:
        raise ValueError(f"x {tuple(x.shape)}, w {tuple(w.shape)}: 1 to {MOST} of each (rows: none, too)")
    _matrix(x, (rows, inner), dev, "x")
    _matrix(w, (cols, inner), dev, "w")
    return rows, inner, cols, dev


def _act_code(act: str) -> int:
    if act not in _ACT:
        raise ValueError(f"act is one of {', '.join(ACTIVATIONS)}, got {act!r}")
    return _ACT[act]


def _padded(t: torch.Tensor) -> bool:
    """Whether a product takes a copy of ``t`` whose rows start on 16-byte boundaries, as tiled loads need it."""
    rows, cols = t.shape
    return t.data_ptr() % 16 != 0 or (rows > 1 and (t.stride(0) % 8 != 0 or t.stride(0) < cols))


def linear_fwd(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, *, act: str = "none",
               resid: torch.Tensor | None = None, keep: bool = False, out: torch.Tensor | None = None,
               z: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``resid + act(x @ w^T + bias)`` for ``x`` [rows, inner] and ``w`` [cols, inner], bf16; ``bias`` [cols] fp32 or bf16 and
    ``resid`` [rows, cols] bf16 may be missing. ``act``: one of :data:`ACTIVATIONS` ("gelu" by the error function, "gelu_tanh" by
    the hyperbolic tangent). Returns (the result, and with ``keep`` the values before the activation, bias included, which
    :func:`linear_bwd` takes: else None). ``out``, ``z``: where to put them; ``out`` may be ``resid`` itself.

    Any sizes and pitches. Rows that start on 16-byte boundaries are fastest: others of ``x`` and ``w`` are copied first, others of
    the results are written element by element."""
    rows, inner, cols, dev = _check(x, w)
    code = _act_code(act)
    if bias is not None and not (bias.shape == (cols,) and bias.dtype in (_F32, _BF16) and bias.device == dev and bias.is_contiguous()):
        raise ValueError(f"bias: contiguous fp32 or bf16 [{cols}] on {dev}, got {_text(bias)}")
    if resid is not None:
        _matrix(resid, (rows, cols), dev, "resid")
    if z is not None and not keep:
        raise ValueError("z is written with keep=True")
    if out is not None:
        _result(out, (rows, cols), dev, "out", x, w, bias, resid, z, inside=resid)
    if z is not None:
        _result(z, (rows, cols), dev, "z", x, w, bias, resid)
    _l.require_cuda(x)
    if out is None:
        out = x.new_empty((rows, cols))
    if keep and z is None:
        z = x.new_empty((rows, cols))
    if rows:
        work, n = None, 0
        pad = _padded(x), _padded(w)
        if pad[0] or pad[1]:
            n = _bytes("aeris_linear_fwd_bytes", rows, inner, cols, *pad)
            work = x.new_empty(n, dtype=torch.uint8)
        _launch("aeris_linear_fwd", _FORWARD.pack(
            x.data_ptr(), w.data_ptr(), 0 if bias is None else bias.data_ptr(), 0 if resid is None else resid.data_ptr(),
            out.data_ptr(), z.data_ptr() if keep else 0, 0 if work is None else work.data_ptr(), _l.status_word(dev).data_ptr(),
            x.stride(0), w.stride(0), 0 if resid is None else resid.stride(0), out.stride(0), z.stride(0) if keep else 0, n,
            rows, inner, cols, code, bias is not None and bias.dtype is _BF16), dev)
    return out, z


def linear_bwd(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, z: torch.Tensor | None = None, *, act: str = "none",
               bias: bool = True, need_dx: bool = True, need_dw: bool = True, dx: torch.Tensor | None = None,
               dw: torch.Tensor | None = None, db: torch.Tensor | None = None):
    """Gradients of :func:`linear_fwd` for ``dy`` [rows, cols] bf16; ``z`` is its second result (not asked for with act="none").
    Returns (gradient of x in bf16 or None, of w in bf16 or None, of the bias in fp32 or, with ``bias=False``, None). The
    gradient of ``resid`` is ``dy``. ``dx``: where to put that of x, not over any input. ``dw`` [cols, inner] and ``db`` [cols], both
    fp32, are added to where given. The same bits on every run.

    The gradient of z is rounded to bf16 for both products; ``db`` sums it before."""
    rows, inner, cols, dev = _check(x, w)
    code = _act_code(act)
    _matrix(dy, (rows, cols), dev, "dy")
    if act != "none":
        if z is None:
            raise ValueError(f"act={act!r}: the backward pass takes z, the values before the activation")
        _matrix(z, (rows, cols), dev, "z")
    else:
        z = None
    if dx is not None and not need_dx or dw is not None and not need_dw or db is not None and not bias:
        raise ValueError("a place for a gradient that is not wanted")
    if dx is not None:
        _result(dx, (rows, inner), dev, "dx", dy, x, w, z, dw, db)
    if dw is not None:
        _result(dw, (cols, inner), dev, "dw", dy, x, w, z, db, dtypes=(_F32,))
    if db is not None:
        if not (db.shape == (cols,) and db.dtype is _F32 and db.device == dev and db.is_contiguous()):
            raise ValueError(f"db: contiguous fp32 [{cols}] on {dev}, got {_text(db)}")
        if any(t is not None and _l.share_memory(db, t) for t in (dy, x, w, z)):
            raise ValueError("db lies over an input")
    _l.require_cuda(x)
    add_db, dw_f32 = db is not None, dw is not None
    make = x.new_empty if rows else x.new_zeros
    if need_dx and dx is None:
        dx = make((rows, inner))
    if need_dw and dw is None:
        dw = make((cols, inner))
    if bias and db is None:
        db = make((cols,), dtype=_F32)
    if rows and (need_dx or need_dw or bias):
        n = _bytes("aeris_linear_bwd_bytes", rows, inner, cols, z is not None or _padded(dy), _padded(x), _padded(w), need_dx, need_dw,
                   bias, dw_f32)
        work = x.new_empty(n, dtype=torch.uint8) if n else None
        _launch("aeris_linear_bwd", _GRAD.pack(
            dy.data_ptr(), x.data_ptr(), w.data_ptr(), 0 if z is None else z.data_ptr(), dx.data_ptr() if need_dx else 0,
            dw.data_ptr() if need_dw else 0, db.data_ptr() if bias else 0, 0 if work is None else work.data_ptr(),
            _l.status_word(dev).data_ptr(), dy.stride(0), x.stride(0), w.stride(0), 0 if z is None else z.stride(0),
            dx.stride(0) if need_dx else 0, dw.stride(0) if need_dw else 0, n, rows, inner, cols, code, dw_f32, add_db), dev)
    return dx, dw, db
