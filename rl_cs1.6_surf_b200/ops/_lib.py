"""ctypes bindings of the CUDA kernel libraries.

Every entry point takes raw device pointers and the CUDA stream to launch on
(the caller's current torch stream), so the kernels compose with torch
tensors and can be captured in CUDA graphs. A non-zero return value is a CUDA
error code and raises.
"""
from __future__ import annotations

import ctypes
from ctypes import c_double, c_float, c_int, c_int64, c_void_p

import numpy as np
import torch

from .._native import load

_V = c_void_p
_I = c_int
_L = c_int64
_F = c_float
_D = c_double

_SIGS = {
    "libsurf_vision.so": {
        "surf_march": (_I, [_V, _L, _I, _I, _I, _V, _I, _I, _I, _F, _F, _F, _F, _V, _V, _F, _F, _I, _I, _V, _L, _I,
                            _I, _V, _V, _I, _V, _V]),
        "surf_brick_size": (_L, [_I, _I, _I]),
        "surf_brick_sdf": (_I, [_V, _I, _V, _I, _I, _I, _V]),
        "surf_brick_i8": (_I, [_V, _V, _I, _I, _I, _V]),
        "surf_occupancy": (_I, [_V, _V, _V, _I, _V, _I, _F, _F, _F, _F, _I, _I, _I, _I, _V, _V]),
        "surf_edt_workspace_bytes": (_L, [_I, _I, _I]),
        "surf_edt": (_I, [_V, _I, _I, _I, _F, _V, _V, _V, _V, _V]),
        "surf_surfnz_bake": (_I, [_V, _I, _V, _V, _V, _I, _V, _I, _D, _D, _D, _D, _I, _I, _I, _V, _V, _V, _V]),
    },
}


class KernelError(RuntimeError):
    pass


_bound: dict = {}


class _Bound:
    """A loaded library exposing only its registered entry points.

    ctypes would call an entry point without a signature by converting every
    Python int to a C int, silently truncating 64-bit device pointers; an
    unregistered name therefore raises instead."""

    def __init__(self, name: str, cdll: ctypes.CDLL):
        self._name = name
        self._cdll = cdll
        for fn, (res, args) in _SIGS.get(name, {}).items():
            f = getattr(cdll, fn)
            f.restype = res
            f.argtypes = args
            setattr(self, fn, f)

    def __getattr__(self, fn: str):
        if fn.startswith("surf_"):
            raise AttributeError(f"{self._name}: entry point {fn} has no registered signature")
        raise AttributeError(fn)


def lib(name: str) -> _Bound:
    if name in _bound:
        return _bound[name]
    b = _Bound(name, load(name))
    _bound[name] = b
    return b


def register(name: str, sigs: dict) -> None:
    _SIGS.setdefault(name, {}).update(sigs)
    _bound.pop(name, None)


def stream_ptr(device=None) -> int:
    return torch.cuda.current_stream(device).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)    # the tensors exist: CUDA is up


def launch(fn, what: str, index: int, *args) -> None:
    """``fn(*args, stream)`` on device ``index`` and its current stream, whatever the
    current device is; raises on a non-zero status."""
    if _current_device() != index:
        with torch.cuda.device(index):
            launch(fn, what, index, *args)
        return
    code = fn(*args, _raw_stream(index) if _raw_stream is not None else stream_ptr(index))
    _launches[0] += _KERNELS_PER_CALL.get(what, 1)
    if code:
        raise KernelError(f"{what} failed with CUDA error {code}")


def ptr(t) -> int:
    return 0 if t is None else int(t.data_ptr())


# Kernel launches issued by each entry point (for launch accounting; entry
# points not listed launch exactly one kernel).
_KERNELS_PER_CALL = {"surf_reward": 2, "surf_permutation": 2, "surf_permutation_pool": 2, "surf_edt": 4, "surf_geodesic_pass": 3,
                     "surf_geodesic_init": 3, "surf_geodesic_finish": 2}
_launches = [0]


def check(code: int, what: str) -> None:
    """Raise on a non-zero CUDA status; count the entry point's launches."""
    _launches[0] += _KERNELS_PER_CALL.get(what, 1)
    if code != 0:
        raise KernelError(f"{what} failed with CUDA error {code}")


def launch_count() -> int:
    """Kernels launched through this package so far (graph replays included
    via ``add_launches``)."""
    return _launches[0]


def add_launches(n: int) -> None:
    _launches[0] += int(n)


def require_cuda(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise KernelError(f"{what}: the CUDA kernel needs CUDA tensors (use the *_reference CPU oracle on CPU)")


class _Extent:
    """Where elements lie, for numpy's overlap test; the memory is never touched."""

    def __init__(self, at: int, size: int, shape, strides):
        self.__array_interface__ = {"version": 3, "typestr": f"|V{size}", "data": (at, False),
                                    "shape": tuple(shape), "strides": tuple(s * size for s in strides)}


def _extent(t: torch.Tensor) -> _Extent:
    return _Extent(t.data_ptr(), t.element_size(), t.shape, t.stride())


def _meet(a: _Extent, b: _Extent) -> bool:
    return bool(np.shares_memory(np.asarray(a), np.asarray(b)))


def _span(t: torch.Tensor) -> tuple:
    """(first address, the one behind the last) of a tensor's elements."""
    at = t.data_ptr()
    if t.is_contiguous():
        return at, at + t.nbytes
    return at, at + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors share an element's memory: exact for strided views, so that
    interleaved columns of one buffer do not count."""
    if not a.numel() or not b.numel():
        return False
    return _meet(_extent(a), _extent(b))


def overlaps_itself(t: torch.Tensor) -> bool:
    """Whether two of a tensor's elements share memory. Exact: by axes from the smallest stride on, whether the axes so
    far meet themselves some steps along the next one, which takes a look only where they reach past its stride."""
    if t.is_contiguous() or t.numel() < 2:
        return False
    at, e, reach = t.data_ptr(), t.element_size(), 0
    axes = sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1)
    for i, (s, n) in enumerate(axes):
        if s == 0:
            return True
        for d in range(1, min(n - 1, reach // s) + 1):
            shape, strides = [m for _, m in axes[:i]], [r for r, _ in axes[:i]]
            if _meet(_Extent(at, e, shape, strides), _Extent(at + d * s * e, e, shape, strides)):
                return True
        reach += (n - 1) * s
    return False


def within_float32(x: float) -> bool:
    """A number that a kernel's float32 argument holds: finite there."""
    return -3.4028234663852886e38 <= x <= 3.4028234663852886e38


def require_apart(what: str, name: str, out: torch.Tensor, inputs: dict, in_place: tuple = ()) -> None:
    """Refuse an ``out`` whose elements share memory with one another or with an input: other
    threads read the inputs while it is written. It may be one of the inputs named in
    ``in_place`` itself, where a thread reads an element before it writes it."""
    lo, hi = _span(out)
    for key, t in inputs.items():
        if not isinstance(t, torch.Tensor):
            continue
        at, end = _span(t)
        if end <= lo or hi <= at:
            continue
        if key in in_place and t.data_ptr() == out.data_ptr() and t.shape == out.shape and t.stride() == out.stride():
            continue
        if overlap(out, t):
            raise ValueError(f"{what}: {name} shares memory with {key}")
    if overlaps_itself(out):
        raise ValueError(f"{what}: {name} has elements that share memory")
