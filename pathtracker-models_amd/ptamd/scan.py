"""Gated linear recurrences (include/pt_scan.h, ``libptscan.so``) and their
autograd bridge.

The framework's cells update their state as ``(1 - g) h + g h^`` (InT / hGRU,
models/InT.py:166,175; the ConvGRU, models/kys.py:46-48) or as ``f c + i tanh(.)``
with an output gate (ConvLSTM, models/convlstm.py:84-90), with gates that look
at the state, so they walk through time.  Where the gates come from the input
alone the same update is linear in the state and can be scanned:

  form     gates, in this order     update (s = logistic function)
  leaky    z, n                     h_t = (1 - s(z_t)) h_{t-1} + s(z_t) n_t;   y_t = h_t
  lstm     i, f, n, o               c_t = s(f_t) c_{t-1} + s(i_t) tanh(n_t);   y_t = s(o_t) tanh(c_t)

``gated_scan`` runs a whole sequence (forward and backward), ``gated_scan_step``
one step of every row in place.  The state is f32 whatever the gates' type
(f32, bf16, f16).  There is no CPU fallback: CPU tensors or a missing library
raise.
"""
from __future__ import annotations

import ctypes
import os
import threading

import torch  # noqa: F401  (its libraries are what _native.so links against)

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libptscan.so")
NATIVE_PATH = os.path.join(HERE, "_native.so")

# Exported symbols declared in include/pt_scan.h (tests check all are present).
EXPORTS = ("pt_scan_backward", "pt_scan_forward", "pt_scan_last_error", "pt_scan_saved_bytes",
           "pt_scan_step", "pt_scan_version", "pt_scan_workspace_bytes")

_P = ctypes.c_void_p
_L = ctypes.c_int64


class Desc(ctypes.Structure):
    _fields_ = [("form", ctypes.c_int32), ("dtype", ctypes.c_int32), ("batch", _L), ("channels", _L),
                ("steps", _L), ("inner", _L)]


class View(ctypes.Structure):
    _fields_ = [("data", _P), ("sb", _L), ("sc", _L), ("st", _L)]


class PtScanError(RuntimeError):
    pass


_lock = threading.RLock()
_lib = None
_native = None


def load():
    """Load (once) and return the C ABI; raise if it is not built."""
    global _lib
    with _lock:
        if _lib is None:
            _require(LIB_PATH)
            lib = ctypes.CDLL(LIB_PATH)
            d, v = ctypes.POINTER(Desc), ctypes.POINTER(View)
            for name in ("pt_scan_saved_bytes", "pt_scan_workspace_bytes"):
                getattr(lib, name).restype = ctypes.c_size_t
                getattr(lib, name).argtypes = [d]
            lib.pt_scan_forward.argtypes = [d, v, _P, _P, v, _P, _P, _P, _P, _P]
            lib.pt_scan_backward.argtypes = [d, v, _P, _P, v, _P, _P, _P, v, _P, _P, _P]
            lib.pt_scan_step.argtypes = [d, v, v, v, _P]
            lib.pt_scan_last_error.restype = ctypes.c_char_p
            lib.pt_scan_version.restype = ctypes.c_char_p
            _lib = lib
    return _lib


def _require(path):
    if not os.path.exists(path):
        raise PtScanError(f"{path} is missing: build the HIP extensions first "
                          "(python __graft_entry__.py build, or python -m ptamd.build)")


def native():
    """The tensors' side (csrc/pt_torch.cpp) on top of the library."""
    global _native
    with _lock:
        if _native is None:
            _require(NATIVE_PATH)
            _require(LIB_PATH)
            from . import _native as mod
            mod.open_scan(LIB_PATH, PtScanError)
            _native = mod
    return _native


def gated_scan(x, h0=None, *, form="leaky", dim=1, gate_dim=2, lengths=None, want_seq=True):
    """The recurrence over a whole sequence, differentiable in the gates and h0 (once,
    and backwards: an input with a forward-mode tangent is refused).

    x: the gates' pre-activations, stacked along ``gate_dim`` of one tensor
      ([B, T, G D] with the defaults; a Conv3d's [B, G C, T, H, W] has dim=2,
      gate_dim=1), or a sequence of G tensors of one shape.  float32, bfloat16
      or float16, any strides; layouts whose last axes are dense are read in
      place, others are copied.
    h0: the state before the first step, a gate's shape without ``dim``
      (None: zeros).
    dim: the time dimension.
    lengths: integer [B] on x's device, B the size of dimension 0: row b ends
      before step lengths[b] (taken into [0, T]).  Nothing behind a row's end is
      read; y and the gradients are 0 there.
    want_seq: False leaves y out (None), where only the last state is used.

    Returns (y, h_last), for lstm (y, h_last, c_last): y in x's type and a
    gate's shape; h_last, f32, is y at each row's last step before its rounding
    (leaky: an empty row keeps h0; lstm: 0 there); c_last, f32, the last state.
    Steps are composed before the state is known: one that becomes infinite may
    be NaN in later steps.
    Forward and backward can be captured into a graph; a captured backward of leaves
    that a graph from the default stream still holds is refused.
    """
    return (_native or native()).gated_scan(x, h0, form, dim, gate_dim, lengths, want_seq)


def gated_scan_step(x, state, *, form="leaky", gate_dim=1):
    """One step of every row: ``state`` (f32, leaky: h, lstm: c) is updated in
    place, y is returned in x's type.

    x: the gates of this step stacked along ``gate_dim`` ([B, G D] with the
      default), or a sequence of G tensors; state: a gate's shape, any strides
      that do not overlap.  No gradients and no tangents: a step that needs a
      backward is a ``gated_scan`` of one step.
    """
    return (_native or native()).gated_scan_step(x, state, form, gate_dim)
