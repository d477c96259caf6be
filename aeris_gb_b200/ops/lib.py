"""ctypes binding of ``libaeris_b200.so`` (C ABI in ``csrc/api.h``).

The library is required on any machine that has a GPU: :func:`lib` raises if it cannot be loaded, so a GPU run can
never silently fall back to the PyTorch reference implementations. On a CPU-only machine the callers use the
pure-PyTorch oracle in :mod:`aeris_gb_b200.models.oracle` instead and never reach this module.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import os

import torch

from .build import LIB_PATH, build, needs_build

_c_int = ctypes.c_int
_c_void_p = ctypes.c_void_p
_c_float = ctypes.c_float
_c_ll = ctypes.c_longlong


class KernelError(RuntimeError):
    pass


@functools.lru_cache(maxsize=None)
def lib() -> ctypes.CDLL:
    if needs_build() and os.environ.get("AERIS_NO_AUTOBUILD") != "1":
        build()
    if not LIB_PATH.exists():
        raise KernelError(f"native library missing: {LIB_PATH}; run `python -m aeris_gb_b200.ops.build`")
    return ctypes.CDLL(str(LIB_PATH))


def ptr(t: torch.Tensor | None) -> _c_void_p:
    return _c_void_p(0 if t is None else t.data_ptr())


def raw_stream() -> int:
    """The current stream of the current device. Asked for on every launch: the raw handle costs 0.3 us, building the
    ``torch.cuda.Stream`` object around it 5 us, a third of what issuing one kernel from Python takes."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def stream_ptr() -> _c_void_p:
    return _c_void_p(raw_stream())


def require_cuda(t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise ValueError(f"the kernels take tensors on a GPU, got one on {t.device}")


_HERE = contextlib.nullcontext()


def on_device(device: torch.device):
    """Context in which ``device`` is the current one."""
    return _HERE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def _pieces(t: torch.Tensor) -> tuple[int, int, list]:
    """(first byte, bytes in one piece, [(how many, bytes apart), ..] from the inside out) of a tensor that is not empty."""
    size = t.element_size()
    width, dims = size, []
    for step, n in sorted((st * size, n) for n, st in zip(t.shape, t.stride()) if n > 1 and st):
        if not dims and step <= width:         # behind one another, or over one another
            width += (n - 1) * step
        elif dims and step == dims[-1][0] * dims[-1][1]:
            dims[-1] = (dims[-1][0] * n, dims[-1][1])
        else:
            dims.append((n, step))
    return t.data_ptr(), width, dims


def share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether ``a`` and ``b`` have a byte in common. Tensors that interleave, such as sections of one matrix's rows, do not. Exact
    where both have one pitch at most and the same one, or the same outermost pitch; two that lie in one range of memory
    otherwise count as sharing it."""
    if not a.numel() or not b.numel():
        return False
    at, wa, da = _pieces(a)
    to, wb, db = _pieces(b)
    if at >= to + wb + sum((n - 1) * s for n, s in db) or to >= at + wa + sum((n - 1) * s for n, s in da):
        return False
    pitches = {d[-1][1] for d in (da, db) if d}
    if len(pitches) != 1 or len(da) > 2 or len(db) > 2:
        return True
    pitch = pitches.pop()
    na, nb = (d[-1][0] if d else 1 for d in (da, db))
    (ma, sa), (mb, sb) = (d[0] if len(d) == 2 else (1, 0) for d in (da, db))
    if sa == sb or mb == 1:
        offsets = range((1 - mb) * sa, ma * sa, sa) if sa else (0,)
    elif ma * mb <= 4096:
        offsets = (i * sa - j * sb for i in range(ma) for j in range(mb))
    else:
        return True
    for d in offsets:
        # pieces r * pitch on in ``a`` and q * pitch on in ``b``, m = r - q: [d + m pitch, .. + wa) against [0, wb)
        d += at - to
        m = max((-wa - d) // pitch + 1, 1 - nb)
        if m < na and d + m * pitch < wb:
            return True
    return False


def same_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether every element of ``a`` lies where the same element of ``b`` does."""
    return (a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.dtype is b.dtype
            and all(n < 2 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride())))


_STATUS: dict[int, torch.Tensor] = {}


def status_word(device: torch.device | None = None) -> torch.Tensor:
    """Per-device int32 word that kernels set when a bounded wait runs out or a bounds check fails; of the current device where
    none is given."""
    dev = torch._C._cuda_getDevice() if device is None else device.index
    if dev not in _STATUS:
        _STATUS[dev] = torch.zeros(1, dtype=torch.int32, device=f"cuda:{dev}")
    return _STATUS[dev]


_ERR_NAMES = {
    1: "timeout waiting for a TMA-filled stage", 2: "timeout waiting for a free stage",
    3: "timeout waiting for an accumulator", 4: "timeout waiting for the epilogue to drain TMEM",
    5: "timeout waiting for a peer signal", 6: "bounds check failed", 7: "timeout inside the attention pipeline",
}


def check_status(sync: bool = True) -> None:
    """Synchronise and raise if any kernel recorded a device-side error since the last check."""
    w = status_word()
    if sync:
        torch.cuda.synchronize()
    code = int(w.item())
    if code != 0:
        w.zero_()
        raise KernelError(f"device-side error {code}: {_ERR_NAMES.get(code, 'unknown')}")


_LAUNCHES = 0


def launch_count() -> int:
    """Number of native kernel launches issued through this module since import."""
    return _LAUNCHES


def check(rc: int, what: str, kernels: int = 1) -> None:
    global _LAUNCHES
    _LAUNCHES += kernels
    if rc != 0:
        raise KernelError(f"{what} failed on the host side with code {rc}")
