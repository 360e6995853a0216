"""Instructions that a whole warp executes are volatile in the sources: an asm without it may be sunk to where its result is used, which may be under a
condition that holds for one lane."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "opfoundry_b200", "csrc")
# exchanges and reductions of a warp, barriers, TMEM loads; products of fragments (mma.sync) stand in straight code whose results all lanes use
WIDE = re.compile(r"redux\.sync|shfl\.sync|vote\.sync|match\.\w+\.sync|elect\.sync|bar\.|barrier\.|tcgen05\.(ld|st|wait|alloc|dealloc|relinquish)")


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.cu*"))), ids=os.path.basename)
def test_warp_wide_instructions_are_volatile(path):
    with open(path) as f:
        text = f.read()
    for m in re.finditer(r"\basm(\s+volatile)?\s*\(((?:\s*\"(?:[^\"\\]|\\.)*\")+)", text):
        if WIDE.search(m.group(2)):
            assert m.group(1), "%s:%d %s" % (os.path.basename(path), text.count("\n", 0, m.start()) + 1, m.group(2).strip()[:60])
