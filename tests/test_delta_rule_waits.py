"""The chunked gated delta rule's kernels wait for one another's warps on mbarriers, whose waits give up after a limit; a
named barrier has none, and a warp that has given up never comes to it."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "delta_feedback_experiment_b200", "csrc")


@pytest.mark.parametrize("name", ["gdr_pairs.cu", "gdr_scan_tc.cu", "gdr_scan_bwd_tc.cu", "gdr_grad_tc.cu", "gdr_tc.cuh"])
def test_no_wait_without_a_limit(name):
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert not re.search(r"\bbar(rier)?\.(cta\.)?sync\b", code)
    assert not re.search(r"\bwhile\b", code)  # (every loop counts)
