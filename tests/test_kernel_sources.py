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
