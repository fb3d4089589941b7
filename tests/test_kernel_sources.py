"""Rules of the kernels' sources that no run shows."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tropical-gemm_b200", "csrc")
FILES = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")))


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_aligned_barriers_meet_whole_warps(path):
    """Barriers that want a warp's lanes together (bar.sync and the aligned cluster barriers) stand behind a __syncwarp()."""
    text = re.sub(r"//.*", "", open(path).read())
    every = re.findall(r'"[^"]*(?:\bbar\.sync|barrier\.cluster\.\w+\.\w+\.aligned)', text)
    safe = re.findall(r'__syncwarp\(\);\s*asm volatile\(\s*"[^"]*(?:\bbar\.sync|barrier\.cluster\.\w+\.\w+\.aligned)', text)
    assert len(every) == len(safe)


def test_a_stage_is_refilled_by_vote():
    """The norm's backward adds up the bytes of rows off the boundaries with an instruction of the whole warp: where a wait before it ran
    out in some of its lanes, none may go on to it, or the others would wait there without a limit."""
    text = open(os.path.join(CSRC, "tg_layernorm.cu")).read()
    assert len(re.findall(r"__reduce_add_sync", text)) == 1 and "if (ACCESS != kAligned) total = __reduce_add_sync(" in text
    waits = re.findall(r"bar_wait\(ring\.empty[^\n]*\n[^\n]*\n[^\n]*", text)
    assert len(waits) == 1
    assert re.search(r"if \(ACCESS != kAligned\) ok = __all_sync\(0xffffffffu, ok\);\n\s*if \(ok\) bring\(", waits[0])
