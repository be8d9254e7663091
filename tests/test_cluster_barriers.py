"""Cluster barriers in their .aligned form are executed by whole warps: behind loops whose lanes leave at different times, too."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "swiftrt_b200", "csrc")


def test_lanes_are_joined_before_an_aligned_cluster_barrier():
    found = 0
    for name in sorted(os.listdir(CSRC)):
        lines = open(os.path.join(CSRC, name)).read().split("\n")
        for i, line in enumerate(lines):
            if re.search(r"barrier\.cluster\.(arrive|wait)[.\w]*\.aligned", line):
                found += 1
                assert "__syncwarp();" in lines[i - 1], f"{name}:{i + 1}"
    assert found
