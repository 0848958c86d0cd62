"""The gated scan against the 64-bit oracle at sizes that bring in each way to cut
time over waves and workgroups.  Which one a size takes shows in the bytes that its
descriptor asks for, so that another rule cannot move a size away unseen."""
import ctypes

import pytest
import torch

from test_gpu_scan import TYPES, _run

pytestmark = pytest.mark.gpu

STEPS = {"leaky": 8, "lstm": 4}           # a wave's steps in a chunk of the backward
FORMS = {"leaky": 0, "lstm": 1}


def _plan(form, dtype, b, c, t, n):
    """(waves, chunks of the backward) of a descriptor; waves 0: a workgroup per chunk."""
    from ptamd import scan
    d = ctypes.byref(scan.Desc(FORMS[form], list(TYPES).index(dtype), b, c, t, n))
    lib = scan.load()
    chunks = lib.pt_scan_saved_bytes(d) // (4 * b * c * n) + 1
    if lib.pt_scan_workspace_bytes(d):
        return 0, chunks
    waves = [w for w in (1, 4, 8, 16) if -(-t // (w * STEPS[form])) == chunks]
    assert len(waves) == 1, waves            # (sizes below tell them apart)
    return waves[0], chunks


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("waves,b,t,f", [(16, 2, 300, 4500), (8, 2, 200, 8300), (4, 600, 70, 60)])
@pytest.mark.parametrize("ragged", [False, True])
def test_waves_of_a_workgroup(form, dtype, waves, b, t, f, ragged):
    ends = None
    if ragged:                               # ends within and between chunks, an empty row
        ends = torch.tensor([t, t - 93] if b == 2 else [(37 * k) % (t + 1) for k in range(b)])
    assert _plan(form, dtype, b, 1, t, f)[0] == waves and _plan(form, dtype, b, 1, t, f)[1] > 1
    assert _plan(form, dtype, 1, b, t, f)[0] == waves        # rows taken as columns
    _run(form, dtype, b, t, f, seed=waves, lengths=ends)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("b,t,f", [(1, 4500, 1024), (16, 4500, 40)])
def test_more_chunks_than_the_card_holds(form, dtype, b, t, f):
    """256 workgroups of 16 waves are at work at a time in the forward, 512 of 8 in the
    backward: the others start when those in front of them end."""
    ends = torch.tensor([(t * (k + 3)) // 18 for k in range(b)]) if b > 1 else None
    waves, chunks = _plan(form, dtype, b, 1, t, f)
    tiles = b * -(-f // 64)
    assert waves == 0 and chunks * tiles > 512 and -(-chunks // 2) * tiles > 256
    _run(form, dtype, b, t, f, seed=t + b, lengths=ends)
