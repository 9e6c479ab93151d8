"""The chunked linear-attention kernel's warps wait for one another on mbarriers, whose waits give up after a limit; a named barrier
has none, and a warp that has given up never comes to it."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "delta_feedback_experiment_b200", "csrc")


def test_no_wait_without_a_limit():
    for name in ("la_tc.cu", "la_tc.cuh"):
        with open(os.path.join(CSRC, name)) as f:
            code = re.sub(r"//[^\n]*", "", f.read())
        assert not re.search(r"\bbar(rier)?\.(cta\.)?sync\b", code)
        assert not re.search(r"\bwhile\b", code)  # (every loop counts)
        assert "kSpinLimit" in code or name.endswith("cuh")


def test_registers_are_given_up_before_they_are_taken():
    """What the warpgroups end up with is what the launch had, or the last of them would wait for good."""
    with open(os.path.join(CSRC, "la_tc.cu")) as f:
        code = f.read()
    v = {m[0]: int(m[1]) for m in re.findall(r"\b(k\w+Regs) = (\d+)", code)}
    assert 256 * v["kStateRegs"] + 128 * v["kOutRegs"] + 256 * v["kOperandRegs"] + 128 * v["kRestRegs"] <= 768 * v["kLaunchRegs"]
    assert all(n % 8 == 0 for n in v.values()) and 768 * v["kLaunchRegs"] <= 65536
