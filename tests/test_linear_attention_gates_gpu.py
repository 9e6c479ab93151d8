"""Linear attention with decays above 1: accepted, and right as long as what they lead to is a number."""

import pytest
import torch

from conftest import assert_close
from linear_attention_cases import FP32_RTOL, HALF_STEP, NAMES, SPLIT, attend, expected, make

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


def recurrent(d):
    from delta_feedback_experiment_b200 import fused_recurrent_linear_attention
    return fused_recurrent_linear_attention(*(d[n] for n in NAMES), initial_state=d["S0"], output_final_state=True)


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
