"""Every loop of the chunked linear-attention kernels has an end that it counts to."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "delta_feedback_experiment_b200", "csrc")


def test_every_loop_has_a_condition():
    with open(os.path.join(CSRC, "la_tc.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert not re.search(r"\b(while|goto|do)\b", code)
    heads = [m.group(1) for m in re.finditer(r"\bfor\s*\(([^;:{}]*;[^;]*;)", code)]
    assert len(heads) > 50
    for head in heads:
        assert head.split(";")[1].strip(), head


def test_a_jump_back_counts_down():
    """The one loop in PTX leaves when its counter is zero, whatever the barrier says."""
    with open(os.path.join(CSRC, "la_tc.cu")) as f:
        code = f.read()
    asm = [a for a in re.findall(r'asm volatile\((.*?)\);', code, re.S) if "bra" in a]
    assert len(asm) == 1
    lines = [line.strip(' "\\nt\t') for line in asm[0].splitlines()]
    text = "\n".join(lines)
    assert re.search(r"mov\.u32 n, %3;.*WAIT_%=:.*sub\.u32 n, n, 1;.*setp\.ne\.u32 q, n, 0;.*@q bra\.uni WAIT_%=;", text, re.S)
    assert text.count("bra") == 2 and "kSpinLimit" in text
