"""Drafted decoding, what needs no GPU: rules that the kernels' sources keep and
arguments at their limits."""

import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rustyneedle_b200", "csrc")


def _kernels():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for body in text.split("__global__")[1:]:
            yield os.path.basename(path), body


def test_no_kernel_reaches_into_a_cluster_before_all_of_it_runs():
    """Another CTA's shared memory may be touched once that CTA is known to run: a cluster barrier comes before the first
    remote access of every kernel that makes one."""
    seen = set()
    for name, body in _kernels():
        first = body.find("map_shared_rank")
        if first < 0:
            continue
        seen.add(name)
        barriers = [body.find(word) for word in ("cluster_wait()", "cluster.sync()") if word in body]
        assert barriers and min(barriers) < first, name
    assert "verify.cu" in seen
