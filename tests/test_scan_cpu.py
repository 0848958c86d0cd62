"""The gated scan's boundary without a GPU: symbols, size queries, refusals of
the C entries (all before any device call) and of ptamd.scan, and how strided
tensors fold into [batch][channels][steps][inner]."""
import ctypes
import os
import re

import pytest
import torch

from ptamd import scan

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_header_binding_and_library_agree():
    txt = open(os.path.join(REPO, "include", "pt_scan.h")).read()
    declared = sorted(set(re.findall(r"\b(pt_scan_[a-z0-9_]+)\s*\(", txt)))
    assert sorted(scan.EXPORTS) == declared
    lib = scan.load()
    assert all(hasattr(lib, s) for s in declared)
    assert lib.pt_scan_version().decode().startswith("pt_scan")


def test_sizes_of_the_buffers():
    lib = scan.load()
    d = scan.Desc(0, 1, 8, 1, 2048, 2048)
    saved = lib.pt_scan_saved_bytes(ctypes.byref(d))
    # one f32 state per chunk of at least 8 steps, none before the first
    assert 0 < saved <= 8 * 2048 * 4 * (2048 // 8 - 1) and saved % (8 * 2048 * 4) == 0
    d.steps = 1
    assert lib.pt_scan_saved_bytes(ctypes.byref(d)) == 0
    assert lib.pt_scan_workspace_bytes(ctypes.byref(d)) == 0
    long = scan.Desc(0, 1, 1, 1, 65536, 64)      # one tile of columns: time is cut over workgroups,
    work = lib.pt_scan_workspace_bytes(ctypes.byref(long))   # a pair of f32 per chunk of 64 steps or more
    assert 0 < work <= 256 + (65536 // 64) * 64 * 8 * 33 // 32


@pytest.mark.parametrize("field,value,word", [
    ("form", 2, b"form"), ("form", -1, b"form"), ("dtype", 3, b"dtype"), ("dtype", -1, b"dtype"),
    ("batch", 0, b">= 1"), ("channels", 0, b">= 1"), ("steps", 0, b">= 1"), ("inner", 0, b">= 1"),
    ("inner", 1 << 29, b"2^29"), ("steps", (1 << 30) + 1, b"2^30"), ("batch", 1 << 60, b"more elements")])
def test_bad_descriptors_are_refused(field, value, word):
    lib = scan.load()
    d = scan.Desc(0, 0, 2, 3, 5, 7)
    setattr(d, field, value)
    one = (scan.View * 4)(*[scan.View(4096, 1, 1, 1) for _ in range(4)])
    assert lib.pt_scan_saved_bytes(ctypes.byref(d)) == 0
    assert word in lib.pt_scan_last_error()
    assert lib.pt_scan_forward(ctypes.byref(d), one, None, None, None, None, None, None, None, None) != 0
    assert lib.pt_scan_backward(ctypes.byref(d), one, None, None, None, None, None, None, one, None, None,
                                None) != 0
    assert lib.pt_scan_step(ctypes.byref(d), one, one, one, None) != 0


def test_bad_pointers_are_refused():
    lib = scan.load()
    d = scan.Desc(0, 0, 1, 1, 100000, 64)
    assert lib.pt_scan_workspace_bytes(ctypes.byref(d)) > 0 and lib.pt_scan_saved_bytes(ctypes.byref(d)) > 0
    good = (scan.View * 4)(*[scan.View(4096, 0, 0, 64) for _ in range(4)])
    null = (scan.View * 4)(scan.View(4096, 0, 0, 64), scan.View(None, 0, 0, 64))
    odd = (scan.View * 4)(*[scan.View(4098, 0, 0, 64) for _ in range(4)])
    r = ctypes.byref(d)

    def fwd(x, work=8192):
        return lib.pt_scan_forward(r, x, None, None, None, None, None, None, work, None)

    apart = (scan.View * 4)(scan.View(4096, 0, 0, 64), scan.View(4096, 0, 0, 128))
    assert fwd(apart) == 2 and b"strides" in lib.pt_scan_last_error()
    for x, work, word in ((None, 8192, b"null"), (null, 8192, b"null"), (good, None, b"workspace"), (good, 8196, b"aligned"),
                          (odd, 8192, b"aligned")):
        assert fwd(x, work) == 1 and word in lib.pt_scan_last_error()
    for saved, work, word in ((None, 8192, b"saved"), (4096, None, b"workspace")):
        assert lib.pt_scan_backward(r, good, None, None, None, None, None, saved, good, None, work, None) == 1
        assert word in lib.pt_scan_last_error()
    assert lib.pt_scan_step(r, good, good, good, None) == 1 and b"steps" in lib.pt_scan_last_error()
    d.steps = 1
    assert lib.pt_scan_step(r, good, None, good, None) == 1 and b"null" in lib.pt_scan_last_error()
    assert lib.pt_scan_step(r, good, odd, good, None) == 1 and b"aligned" in lib.pt_scan_last_error()


def test_refusals_of_tensors():
    x = torch.zeros(2, 5, 8)
    with pytest.raises(ValueError, match="form"):
        scan.gated_scan(x, form="gru")
    with pytest.raises(ValueError, match="multiple"):
        scan.gated_scan(torch.zeros(2, 5, 7))
    with pytest.raises(ValueError, match="dimensions"):
        scan.gated_scan(torch.zeros(2, 8), gate_dim=1)
    with pytest.raises(ValueError, match="gate_dim"):
        scan.gated_scan(x, gate_dim=3)
    with pytest.raises(ValueError, match="gates"):
        scan.gated_scan([x, x, x])
    with pytest.raises(ValueError, match="one shape"):
        scan.gated_scan([x, x[:, :4]])
    with pytest.raises(TypeError, match="type"):
        scan.gated_scan(x.double())
    with pytest.raises(TypeError, match="one type"):
        scan.gated_scan([x, x.bfloat16()])
    with pytest.raises(TypeError, match="tensors"):
        scan.gated_scan([x, 1.0])
    with pytest.raises(scan.PtScanError, match="ROCm device"):      # no CPU fallback
        scan.gated_scan(x)
    with pytest.raises(scan.PtScanError, match="ROCm device"):
        scan.gated_scan_step(torch.zeros(2, 8), torch.zeros(2, 4))


def _index(fold, shape, dim, strides, which, at):
    """Offset that the fold gives the element ``at`` of tensor ``which``."""
    b, c, n, each = fold
    sb, sc, st = each[which]
    rest = [k for k in range(len(shape)) if k != dim]
    flat = 0
    for k in rest:
        flat = flat * shape[k] + at[k]
    bi, ci, ni = flat // (c * n), flat // n % c, flat % n
    return bi * sb + ci * sc + ni + (0 if dim is None else at[dim] * st)


@pytest.mark.parametrize("shape,dim,perms,batch_first", [
    ((2, 5, 6), 1, [None, None], True),
    ((2, 5, 6), 2, [None, (2, 0, 1)], True),
    ((5, 2, 6), 0, [None, (1, 0, 2)], False),
    ((2, 3, 4, 5, 6), 2, [None], True),
    ((2, 3, 4, 5, 6), 2, [(0, 2, 1, 3, 4), None], True),
    ((2, 3, 4, 5, 6), 1, [None, (0, 1, 2, 3, 4)], True),
    ((1, 3, 1, 5, 1), 1, [None], True),
    ((4, 6), None, [None, (1, 0)], False),
    ((4, 3, 5), None, [None, None, None], False),
])
def test_fold_addresses_every_element(shape, dim, perms, batch_first):
    tensors = []
    for p in perms:
        if p is None:
            tensors.append(torch.empty(shape))
        else:                                   # memory order p, axes back in place
            t = torch.empty([shape[k] for k in p])
            tensors.append(t.permute([p.index(k) for k in range(len(shape))]))
    strides = tuple(t.stride() for t in tensors)
    fold = scan.native().fold(shape, -1 if dim is None else dim, strides, batch_first)
    if fold is None:
        assert any(p is not None for p in perms)      # dense tensors of one order always fold
        return
    assert fold[0] * fold[1] * fold[2] * (1 if dim is None else shape[dim]) == torch.empty(shape).numel()
    if batch_first and dim != 0:
        assert fold[0] == shape[0]
    for k, st in enumerate(strides):
        for at in torch.cartesian_prod(*[torch.arange(n) for n in shape]).reshape(-1, len(shape)).tolist():
            assert _index(fold, shape, dim, strides, k, at) == sum(a * s for a, s in zip(at, st))


def test_fold_refuses_what_it_cannot_address():
    # three separately strided groups in front of a dense axis
    t = torch.empty(2, 3, 4, 5, 6).permute(0, 2, 1, 3, 4)
    strided = torch.empty(4, 6, 8, 5, 6)[::2, ::2, ::2]
    assert scan.native().fold((2, 3, 4, 5, 6), 3, (strided.stride(),), True) is None
    assert scan.native().fold(t.shape, 3, (t.stride(),), True) is None


def test_overlapping_states_are_seen():
    apart = scan.native().disjoint
    assert apart((4, 6), (6, 1)) and apart((4, 6), (1, 4)) and apart((1, 6), (0, 1)) and apart((4, 6), (100, 2))
    assert not apart((4, 6), (0, 1)) and not apart((4, 6), (3, 1))


def test_fold_keeps_the_batch_apart():
    """Row ends are read per batch row, and how the columns are cut decides where the
    backward finds its states: no layout may take another axis into the batch."""
    fold = scan.native().fold
    # memory [T][B][P][Q + 1][N + 1]: B and P lie like one axis, P and Q do not
    x = torch.empty(5, 4, 6, 6, 9)[:, :, :, :5, :8].transpose(0, 1)          # [B, T, P, Q, N]
    assert fold(x.shape, 1, (x.stride(),), True) is None
    dense = torch.empty(x.shape)
    assert fold(x.shape, 1, (dense.stride(),), True)[0] == 4
    # time first: the batch and P apart in one tensor, together in another
    y = torch.empty(5, 4, 7, 9)[:, :, :6, :8]
    assert fold(y.shape, 0, (y.stride(),), False) is None
    assert fold(y.shape, 0, (torch.empty(y.shape).stride(),), False)[:2] == (1, 1)
    # a step has neither: its columns may be cut anyhow
    assert fold((4, 6, 5, 8), -1, (x.select(1, 0).stride(),), -1)[0] == 24


def test_more_threads_than_a_launch_takes_are_refused():
    """Before anything is launched (a launch fails differently here, without a device)."""
    lib = scan.load()
    one = (scan.View * 4)(*[scan.View(4096, 0, 0, 0) for _ in range(4)])
    ends = 4096

    def rc(*desc):
        d = scan.Desc(*desc)
        out = [lib.pt_scan_forward(ctypes.byref(d), one, None, ends, None, None, None, None, 8192, None),
               lib.pt_scan_backward(ctypes.byref(d), one, None, ends, None, None, None, 4096, one, None, 8192, None)]
        return out, lib.pt_scan_last_error()

    for desc in ((0, 1, 1, 1, 1 << 30, 1), (1, 1, 1, 1, 1 << 29, 64),          # chunks of one long row
                 (0, 1, 1 << 24, 1, 100, 1), (1, 0, 1 << 26, 1, 4, 3)):        # rows, four waves and one
        codes, word = rc(*desc)
        assert codes == [2, 2] and b"launch takes" in word, (desc, codes, word)
    d = scan.Desc(0, 0, 1 << 32, 1, 1, 1)
    assert lib.pt_scan_step(ctypes.byref(d), one, one, one, None) == 2 and b"launch takes" in lib.pt_scan_last_error()
