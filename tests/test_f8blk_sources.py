"""The bounded waits of the block-scaled e4m3 kernels as the sources write them: given up by the whole warp, and named barriers that every
warp still comes to.  The case itself cannot be made on a GPU without hanging it, so this reads the sources."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paddock_b200", "csrc")


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


@pytest.mark.parametrize("name,least", [("f8blk_split.cu", 4), ("f8blk_wide.cu", 5)])
def test_a_wait_is_given_up_by_the_whole_warp(name, least):
    text = source(name)
    assert not re.search(r"\bmbar_wait\(", text)
    found = [m for m in re.finditer(r"\bwait_soon\(", text)]
    assert len(found) >= least
    for m in found:
        start = max(text.rfind(c, 0, m.start()) for c in ";{}")
        end = text.index(";", text.index(";", m.end()) + 1)
        assert "__all_sync(0xffffffffu" in text[start:end], text[start:end]


def test_warps_that_gave_up_still_come_to_the_named_barriers():
    """The wide kernel's product warps meet twice per tile of the gated front; nothing leaves their loop over tiles."""
    text = source("f8blk_wide.cu")
    loop = text[text.index("for (uint32_t tile = blockIdx.x; tile < n_tiles; tile += gridDim.x)"):]
    loop = loop[:loop.index("\n        }\n")]
    assert loop.count("bar.sync 1, 256;") == 2 and "return" not in loop.replace("return more", "")
    blocks = loop[loop.index("for (uint32_t kb = 0"):loop.index("if constexpr (kPlanes == 1)")]
    assert loop.count("break;") == blocks.count("break;") == 1          # it leaves the loop over blocks of K only
    assert "ok" in loop[loop.index("bar.sync"):]                        # and nothing is stored behind a wait that ran out
