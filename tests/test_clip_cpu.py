"""Gradient clipping's boundary without a GPU: symbols, refusals of the C
entries (before any device call) and of ptamd.clip."""
import ctypes
import os
import re

import pytest
import torch

from ptamd import clip

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_header_binding_and_library_agree():
    txt = open(os.path.join(REPO, "include", "pt_clip.h")).read()
    declared = sorted(set(re.findall(r"\b(pt_clip_[a-z0-9_]+)\s*\(", txt)) - {"pt_clip_tensor"})
    assert sorted(clip.EXPORTS) == declared
    lib = clip.load()
    assert all(hasattr(lib, s) for s in declared)
    assert lib.pt_clip_version().decode().startswith("pt_clip")


def _table(*rows):
    return (clip.Tensor * len(rows))(*rows)


def test_workspace_grows_with_the_tensors_and_stays_small():
    lib = clip.load()
    one = _table((1 << 20, 1 << 20, 5, 0, 0))
    assert lib.pt_clip_workspace_bytes(one, 1) == 16
    assert lib.pt_clip_workspace_bytes(_table((None, None, 0, 0, 0)), 1) == 8
    big = _table(*[(1 << 20, 1 << 20, 1 << 27, 1, 1)] * 1000)
    assert 8 < lib.pt_clip_workspace_bytes(big, 1000) <= 1 << 20


@pytest.mark.parametrize("row,word", [
    ((1 << 20, 1 << 20, -1, 0, 0), b"negative"),
    ((1 << 20, 1 << 20, 1 << 45, 0, 0), b"2^44"),
    ((1 << 20, 1 << 20, 4, 3, 0), b"type"),
    ((None, 1 << 20, 4, 0, 0), b"null"),
    ((1 << 20, None, 4, 0, 0), b"null"),
    (((1 << 20) + 2, 1 << 20, 4, 0, 0), b"aligned"),
    ((1 << 20, (1 << 20) + 2, 4, 1, 0), b"aligned"),
    ((1 << 20, 1 << 20, 4, 0, 1), b"f32"),
    ((1 << 20, 1 << 20, 4, 1, 2), b"f32"),
    ((1 << 20, 1 << 20, 4, 1, 0), b"shares memory"),            # widened over its own input
    ((1 << 20, (1 << 20) + 4, 4, 0, 0), b"shares memory"),      # shifted over its own input
])
def test_bad_tensors_are_refused(row, word):
    lib = clip.load()
    assert lib.pt_clip_grads(_table(row), 1, 2, 1.0, 4096, 4096, None) in (1, 2)
    assert word in lib.pt_clip_last_error(), lib.pt_clip_last_error()


def test_shared_memory_is_refused():
    lib = clip.load()
    a = 1 << 20

    def refused(*rows):
        rc = lib.pt_clip_grads(_table(*rows), len(rows), 2, 1.0, 4096, 4096, None)
        return rc == 1 and b"shares memory" in lib.pt_clip_last_error()

    assert refused((a, a, 8, 0, 0), (a, a, 8, 0, 0))                       # the same tensor twice
    assert refused((a, a, 8, 0, 0), (a + 28, a + 28, 8, 0, 0))             # the last element
    assert refused((a, a + 4096, 8, 0, 0), (a + 64, a + 4096, 8, 0, 0))    # one output for two
    assert refused((a, a + 64, 8, 0, 0), (a + 64, a + 4096, 8, 0, 0))      # an output over the next input
    assert refused((a, a, 100, 0, 0), (a + 4, a + 4, 1, 0, 0), (a + 4096, a + 4096, 1, 0, 0))


def test_bad_calls_are_refused():
    lib = clip.load()
    one = _table((1 << 20, 1 << 20, 5, 0, 0))
    for bad in (-1.0, float("nan")):
        assert lib.pt_clip_grads(one, 1, 2, bad, 4096, 4096, None) == 1
        assert b"max_norm" in lib.pt_clip_last_error()
    assert lib.pt_clip_grads(one, 1, 3, 1.0, 4096, 4096, None) == 1 and b"norm" in lib.pt_clip_last_error()
    assert lib.pt_clip_grads(one, 1, 2, 1.0, None, 4096, None) == 1 and b"null" in lib.pt_clip_last_error()
    assert lib.pt_clip_norm(one, 1, 2, 4096, None, None) == 1 and b"null" in lib.pt_clip_last_error()
    assert lib.pt_clip_norm(None, 1, 2, 4096, 4096, None) == 1 and b"null" in lib.pt_clip_last_error()


def test_python_refusals():
    g = torch.zeros(4)
    with pytest.raises(clip.PtClipError, match="ROCm device"):      # no CPU fallback
        clip.clip_grads([g], 1.0)
    with pytest.raises(TypeError, match="type"):
        clip.grad_norm([g.double()])
    with pytest.raises(ValueError, match="max_norm"):
        clip.clip_grads([g], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip.clip_grads([g], float("nan"))
    with pytest.raises(ValueError, match="norm_type"):
        clip.grad_norm([g], 3)
    with pytest.raises(ValueError, match="outputs"):
        clip.clip_grads([g], 1.0, out=[])
    assert float(clip.clip_grads([], 1.0)) == 0.0
    p = torch.nn.Parameter(torch.zeros(3))                          # no gradient: left out
    assert float(clip.clip_grad_norm_([p], 1.0)) == 0.0

