"""Linear attention with decays above 1: accepted, and right as long as what they lead to is a number."""

import pytest
import torch

from conftest import assert_close, rel_rms
from linear_attention_cases import FP32_RTOL, HALF_STEP, NAMES, SPLIT, attend, check, expected, make, run_with_grads
from linear_attention_chunks64 import attend_with_grads as chunks64

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


def recurrent(d):
    from delta_feedback_experiment_b200 import fused_recurrent_linear_attention
    return fused_recurrent_linear_attention(*(d[n] for n in NAMES), initial_state=d["S0"], output_final_state=True)


def fall_and_rise(d, steps):
    """Log-decays at single tokens; what happens while the state is small neither writes nor is written to, so that every result
    stays in the range of the others."""
    d["g"].fill_(-0.01)
    for t, x in steps:
        d["g"][:, t] = x
    first, last = steps[0][0], steps[-1][0]
    for n in ("k", "v"):
        d[n][:, first:last] = 0
    return d


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (FP32, 64)])
@pytest.mark.parametrize("steps", [[(20, -80.0), (30, 80.0)], [(10, -40.0), (11, -40.0), (63, 79.0)], [(70, -50.0), (90, -30.0), (100, 45.0), (101, 35.0)],
                                   [(40, -55.0), (90, 55.0)]],
                         ids=["once", "to the chunk's end", "in steps", "over chunks"])
def test_a_decay_that_is_taken_back(dtype, D, steps):
    d = fall_and_rise(make(1, 150, 1, 2, D, dtype, 31), steps)
    got, want = run_with_grads(d), expected(d)
    if dtype == FP32 and min(sum(x for _, x in steps[:i + 1]) for i in range(len(steps))) < -70:
        # Token by token a state of 0.3 is at 2^-117 behind e^-80, where numbers end at 2^-126: each entry is off by that, 2^-10.6
        # when it is back; a product of 64 of them with a row of length 1 by 8 times that at most, 2^-5.9 of 0.3.
        for n, t in got.items():
            assert_close(t, want[n], 2.0 ** -5.9, n, outlier_frac=0.0)
        return
    check(got, want, d)


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("HV", [2, 160], ids=["side by side", "walked"])
@pytest.mark.parametrize("down,up", [(100, 400), (400, 100), (200, 1200), (1200, 200)])
def test_a_decay_that_is_taken_back_in_another_segment(D, HV, down, up):
    """A segment is 256 to 1,024 tokens.  Between the two tokens nothing is written, read or asked for: the gradients there are of what
    passes over, which is as large as elsewhere."""
    d = make(1, max(down, up) + 150, 1, HV, D, BF16, 36)
    d["g"].fill_(-0.002)
    d["g"][:, down], d["g"][:, up] = -55.0, 55.0
    first, last = min(down, up), max(down, up)
    for n in ("q", "k", "v", "do"):
        d[n][:, first:last] = 0
    check(run_with_grads(d), chunks64(d), d)


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("HV", [2, 160], ids=["side by side", "walked"])
@pytest.mark.parametrize("gates", [(-55.0, 50.0, 50.0, -45.0), (50.0, -55.0, -35.0, 40.0), (45.0, -55.0, -55.0, 65.0)],
                         ids=["grows", "decays", "leaves its range"])
def test_a_segment_beyond_the_range_of_one_number(D, HV, gates):
    """Each chunk's decay is a number, and so are the states: a segment's, 2^144, 2^-130 or 2^-159, need not be."""
    d = make(1, 700, 1, HV, D, BF16, 37)
    d["g"].fill_(-0.002)
    for t, x in zip((100, 300, 400, 600), gates):
        d["g"][:, t] = x
    for n in ("q", "k", "v", "do"):
        d[n][:, 100:600] = 0
    got, want = run_with_grads(d), chunks64(d)
    if gates[-1] == 65.0:
        # What passes over is at 2^-94.9 of what it was and will be (65 units of log e and 1.1 of the other tokens'), below the stated 2^-85.
        # The kernels hold it in units of 2^24, where numbers end at 2^-126: an entry is off by 2^-7.1 at most when it is back, 2^-5.4 of
        # the 0.3 that entries are, and so are, in the mean, products with rows of length 1.
        for n, t in got.items():
            assert rel_rms(t, want[n]) <= 2.0 ** -5.4, n
        return
    check(got, want, d)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (FP32, 32)])
@pytest.mark.parametrize("top", [0.05, 0.6])
def test_gates_of_both_signs(dtype, D, top):
    d = make(2, 200, 1, 2, D, dtype, 32)
    gen = torch.Generator().manual_seed(33)
    d["g"] = (top * (2 * torch.rand(d["g"].shape, generator=gen) - 1)).cuda()
    check(run_with_grads(d), expected(d), d)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (FP32, 64), (FP32, 8)])
def test_the_largest_decays(dtype, D):
    """e^88.5 = 2^127.7 is a number; from 2^128 on no decay of a token is one (in chunks what counts is what it does together with its
    neighbours', up to a gate of 128, which no number follows)."""
    d = make(1, 2, 1, 2, D, dtype, 34)
    d["g"][:, 0] = -1.0
    d["g"][:, 1, 0], d["g"][:, 1, 1] = 88.5, 60.0
    d["S0"] *= 1e-3
    for n in ("v", "k"):
        d[n][:, 0] *= 2.0 ** -8
    d["q"][:, 1] *= 2.0 ** -10
    want = expected(d)
    for o, S in (recurrent(d), attend(d)):
        chunked = dtype == BF16
        assert_close(S, want["S"], SPLIT if chunked else FP32_RTOL, "S")
        assert_close(o, want["o"], (SPLIT + HALF_STEP) if chunked else FP32_RTOL, "o")
    for g in (89.0, 1e30, float("inf")):
        d["g"][:, 1, 0] = g
        for o, S in [recurrent(d)] + ([attend(d)] if g > 128 or dtype == FP32 else []):
            assert not S[:, 0].isfinite().any() and not o[:, 1, 0].isfinite().any()
            assert_close(S[:, 1], want["S"][:, 1], SPLIT if chunked else FP32_RTOL, "S")
