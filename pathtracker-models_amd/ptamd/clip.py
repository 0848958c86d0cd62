"""The global gradient norm and clipping (include/pt_clip.h, ``libptclip.so``).

The reference's ``clip_grad_norm_`` (utils/misc_functions.py:48-69) over any
number of tensors in two launches for every 192 to 320 of them, with sums in 64 bits
and a fixed order of addition, so that data-parallel ranks that hold the same
averaged gradients clip them by the same factor bit for bit.  The norm stays on
the device: nothing here synchronises, unless ``error_if_nonfinite`` asks.
There is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math
import os
import threading

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libptclip.so")
NATIVE_PATH = os.path.join(HERE, "_native.so")

# Exported symbols declared in include/pt_clip.h (tests check all are present).
EXPORTS = ("pt_clip_grads", "pt_clip_last_error", "pt_clip_norm", "pt_clip_version",
           "pt_clip_workspace_bytes")

_P = ctypes.c_void_p


class Tensor(ctypes.Structure):
    _fields_ = [("grad", _P), ("out", _P), ("n", ctypes.c_int64), ("grad_type", ctypes.c_int32),
                ("out_type", ctypes.c_int32)]


class PtClipError(RuntimeError):
    pass


_lock = threading.RLock()
_lib = None
_native = None


def _require(path):
    if not os.path.exists(path):
        raise PtClipError(f"{path} is missing: build the HIP extensions first "
                          "(python __graft_entry__.py build, or python -m ptamd.build)")


def load():
    """Load (once) and return the C ABI; raise if it is not built."""
    global _lib
    with _lock:
        if _lib is None:
            _require(LIB_PATH)
            lib = ctypes.CDLL(LIB_PATH)
            t = ctypes.POINTER(Tensor)
            lib.pt_clip_workspace_bytes.restype = ctypes.c_size_t
            lib.pt_clip_workspace_bytes.argtypes = [t, ctypes.c_int64]
            lib.pt_clip_norm.argtypes = [t, ctypes.c_int64, ctypes.c_int, _P, _P, _P]
            lib.pt_clip_grads.argtypes = [t, ctypes.c_int64, ctypes.c_int, ctypes.c_double, _P, _P, _P]
            lib.pt_clip_last_error.restype = ctypes.c_char_p
            lib.pt_clip_version.restype = ctypes.c_char_p
            _lib = lib
    return _lib


def native():
    """The tensors' side (csrc/pt_torch.cpp) on top of the library."""
    global _native
    with _lock:
        if _native is None:
            _require(NATIVE_PATH)
            _require(LIB_PATH)
            from . import _native as mod
            mod.open_clip(LIB_PATH, PtClipError)
            _native = mod
    return _native


def grad_norm(grads, norm_type=2.0):
    """The norm of all elements of the tensors together: f32, a device scalar
    (of no tensors: 0, on the CPU)."""
    norm = (_native or native()).clip(list(grads), norm_type, -1.0, None)
    return torch.zeros(()) if norm is None else norm


def clip_grads(grads, max_norm, *, norm_type=2.0, out=None):
    """Scale the tensors together to a norm of at most ``max_norm``; returns the
    norm before (f32, a device scalar; of no tensors: 0, on the CPU).

    grads: tensors of float32, bfloat16 or float16 (mixed, empty ones too) on
      one device, sharing no memory with each other; no forward-mode tangents.
    out: None scales in place; else one tensor per gradient, of its shape and of
      its type or float32 (an optimizer's f32 buffers for 16-bit gradients).
    norm_type: 1, 2 or inf.
    """
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm {max_norm} must be >= 0")
    norm = (_native or native()).clip(list(grads), norm_type, max_norm, None if out is None else list(out))
    return torch.zeros(()) if norm is None else norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Clip the gradients of ``parameters`` (one or several) in place; returns
    their norm before (reference utils/misc_functions.py:48-69).  Parameters
    without a gradient are left out; one listed twice is refused (its gradient
    would be scaled twice)."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads, norm_type = [p.grad for p in parameters if p.grad is not None], float(norm_type)
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"the gradients' norm is {float(norm)}: nothing was clipped")
    return clip_grads(grads, max_norm, norm_type=norm_type)
