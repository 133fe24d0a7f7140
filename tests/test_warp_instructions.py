"""Instructions that all lanes of a warp take part in are volatile in the kernels' sources: the compiler may move one that is not under divergent code."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rustane_b200", "csrc")


def test_whole_warp_instructions_are_volatile():
    seen = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = open(path).read()
        for at in re.finditer(r'\basm\b(\s+volatile)?\s*\(\s*"([^"]*)', text):
            if re.search(r"mma\.sync|ldmatrix|stmatrix|bar\.sync|\.sync\.aligned", at.group(2)):
                seen += 1
                assert at.group(1), "%s: %s" % (os.path.basename(path), at.group(2))
    assert seen >= 6
