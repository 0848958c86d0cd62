"""tools/isa_listing.py leaves the library that it lists as it is: the process
that lists it may have it loaded."""
import hashlib
import importlib
import os
import re
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_listing_does_not_touch_the_library():
    sys.path.insert(0, os.path.join(REPO, "tools"))
    import isa_listing
    from ptamd import clip
    before = os.stat(clip.LIB_PATH)
    digest = hashlib.sha256(open(clip.LIB_PATH, "rb").read()).hexdigest()
    assert ".Lfunc_end" in isa_listing.listing(clip.LIB_PATH)
    after = os.stat(clip.LIB_PATH)
    assert (before.st_ino, before.st_mtime_ns) == (after.st_ino, after.st_mtime_ns)
    assert hashlib.sha256(open(clip.LIB_PATH, "rb").read()).hexdigest() == digest


@pytest.mark.parametrize("lib", ["scan", "clip"])
def test_no_packed_f32_arithmetic_and_no_scratch_memory(lib):
    """The scan's and the clipping's libraries are built without packed-FP32
    instructions; and no kernel keeps values in scratch memory (an array there added
    a seventh to what the backward writes)."""
    sys.path.insert(0, os.path.join(REPO, "tools"))
    import isa_listing
    text = isa_listing.disassemble(importlib.import_module(f"ptamd.{lib}").LIB_PATH)
    assert re.search(r"\bv_fma", text)
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
    assert not re.search(r"\bscratch_(store|load)", text)
