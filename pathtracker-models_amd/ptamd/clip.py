"""The global gradient norm and clipping (include/pt_clip.h, ``libptclip.so``).

The reference's ``clip_grad_norm_`` (utils/misc_functions.py:48-69) over any
number of tensors in two launches for every 96 of them, with sums in 64 bits
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

from .scan import _on

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libptclip.so")

# Exported symbols declared in include/pt_clip.h (tests check all are present).
EXPORTS = ("pt_clip_grads", "pt_clip_last_error", "pt_clip_norm", "pt_clip_version",
           "pt_clip_workspace_bytes")

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_NORMS = {math.inf: 0, 1.0: 1, 2.0: 2}
_P = ctypes.c_void_p


class Tensor(ctypes.Structure):
    _fields_ = [("grad", _P), ("out", _P), ("n", ctypes.c_int64), ("grad_type", ctypes.c_int32),
                ("out_type", ctypes.c_int32)]


class PtClipError(RuntimeError):
    pass


_lock = threading.RLock()
_lib = None


def load():
    """Load (once) and return the library; raise if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise PtClipError(f"{LIB_PATH} is missing: build the HIP extensions first "
                                  "(python __graft_entry__.py build, or python -m ptamd.build)")
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


def _chk(lib, rc):
    if rc != 0:
        raise PtClipError(f"pt_clip error {rc}: {lib.pt_clip_last_error().decode(errors='replace')}")


def _norm_code(norm_type):
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type {norm_type!r}: 1, 2 or inf")
    return code


def _dense(t):
    """Whether every element is at a place of its own and the places are one run:
    then the order of the axes does not matter here."""
    if t.is_contiguous():
        return True
    run = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if st != run:
            return False
        run *= n
    return True


def _check(tensors, what):
    dev = None
    for t in tensors:
        if not isinstance(t, torch.Tensor) or t.layout is not torch.strided:
            raise TypeError(f"{what} must be dense tensors")
        if t.dtype not in _TYPES:
            raise TypeError(f"{what} of type {t.dtype}: float32, bfloat16 or float16")
        if not t.is_cuda:
            raise PtClipError("clipping runs on a ROCm device only (no CPU fallback)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise PtClipError(f"{what} are on several devices ({dev}, {t.device}): one process per GPU")
    return dev


def _run(grads, norm_type, max_norm=None, out=None):
    code = _norm_code(norm_type)
    dev = _check(grads, "gradients")
    if dev is None:
        return torch.zeros(()) if not torch.cuda.is_available() else torch.zeros((), device="cuda")
    lib = load()
    back = []                                    # (tensor, dense copy): outputs to copy back
    src = [g if _dense(g) else g.contiguous() for g in grads]
    if max_norm is None:
        dst = src
    elif out is None:
        dst = src
        for g, s in zip(grads, src):
            if s is not g:
                if any(st == 0 and n > 1 for st, n in zip(g.stride(), g.shape)):
                    raise PtClipError("a gradient's elements share memory (an expanded tensor): "
                                      "it cannot be clipped in place")
                back.append((g, s))
    else:
        dst = []
        for g, s, o in zip(grads, src, out):
            if o is g:
                if s is not g:
                    back.append((g, s))
                dst.append(s)
            elif o.stride() == s.stride() and _dense(o):
                dst.append(o)
            else:                                # another order of the axes: through a copy
                d = torch.empty_like(s, dtype=o.dtype)
                back.append((o, d))
                dst.append(d)
    n = len(src)
    table = (Tensor * n)(*[(s.data_ptr(), d.data_ptr(), s.numel(), _TYPES[s.dtype], _TYPES[d.dtype])
                           for s, d in zip(src, dst)])
    with _on(dev) as stream:
        size = lib.pt_clip_workspace_bytes(table, n)
        if size == 0:
            _chk(lib, 1)
        work = torch.empty(size, dtype=torch.uint8, device=dev)
        norm = torch.empty((), device=dev)
        if max_norm is None:
            _chk(lib, lib.pt_clip_norm(table, n, code, norm.data_ptr(), work.data_ptr(), stream))
        else:
            _chk(lib, lib.pt_clip_grads(table, n, code, max_norm, norm.data_ptr(), work.data_ptr(), stream))
    for o, d in back:
        o.copy_(d)
    return norm


@torch.no_grad()
def grad_norm(grads, norm_type=2.0):
    """The norm of all elements of the tensors together: f32, a device scalar."""
    return _run(list(grads), norm_type)


@torch.no_grad()
def clip_grads(grads, max_norm, *, norm_type=2.0, out=None):
    """Scale the tensors together to a norm of at most ``max_norm``; returns the
    norm before (f32, a device scalar).

    grads: tensors of float32, bfloat16 or float16 (mixed, empty ones too) on
      one device, sharing no memory with each other.
    out: None scales in place; else one tensor per gradient, of its shape and of
      its type or float32 (an optimizer's f32 buffers for 16-bit gradients).
    norm_type: 1, 2 or inf.
    """
    grads = list(grads)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm {max_norm} must be >= 0")
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"{len(out)} outputs for {len(grads)} gradients")
        dev = _check(grads, "gradients")
        if out and _check(out, "outputs") != dev:
            raise PtClipError("outputs are not on the gradients' device")
        for g, o in zip(grads, out):
            if o.shape != g.shape:
                raise ValueError(f"an output of shape {tuple(o.shape)} for a gradient of shape {tuple(g.shape)}")
            if o.dtype not in (g.dtype, torch.float32):
                raise TypeError(f"an output of type {o.dtype} for a gradient of type {g.dtype}")
    return _run(grads, norm_type, max_norm, out)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Clip the gradients of ``parameters`` (one or several) in place; returns
    their norm before (reference utils/misc_functions.py:48-69).  Parameters
    without a gradient are left out."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"the gradients' norm is {float(norm)}: nothing was clipped")
    return clip_grads(grads, max_norm, norm_type=norm_type)
