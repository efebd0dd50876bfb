"""CPU checks of the kernels' sources."""
from __future__ import annotations

import glob
import os
import re

CSRC = os.path.join(os.path.dirname(__file__), "..", "moonxi-net_b200", "csrc")


def _sources():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        with open(path) as f:
            yield os.path.basename(path), f.read().splitlines()


def test_lanes_meet_before_a_named_barrier():
    """bar.sync is barrier.sync.aligned: one instruction of all 32 lanes, too."""
    checked = 0
    for name, lines in _sources():
        for i, line in enumerate(lines):
            if '"bar.sync' in line.split("//")[0]:
                checked += 1
                assert any("__syncwarp()" in x for x in lines[max(0, i - 4):i]), (name, i + 1)
    assert checked >= 2


def test_lanes_meet_before_a_warps_collective_instructions():
    """A TMEM load and a cluster barrier (.aligned) are one instruction of all 32
    lanes.  Their lanes part in the loops and branches before them (rows past the
    last one, an activation's cases), so each has a __syncwarp() close before it."""
    checked = 0
    for name, lines in _sources():
        for i, line in enumerate(lines):
            code = line.split("//")[0]
            if re.search(r"(?<!void )tmem_ld_32cols\(", code) or "barrier.cluster.arrive" in code:
                checked += 1
                assert any("__syncwarp()" in x for x in lines[max(0, i - 4):i]), (name, i + 1)
    assert checked >= 3
