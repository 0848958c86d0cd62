"""tools/isa_listing.py leaves the library that it lists as it is: the process
that lists it may have it loaded."""
import hashlib
import os
import sys

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
