"""The range of numbers that linear attention takes."""

import pytest
import torch

from linear_attention_cases import NAMES, attend, check, make, run_with_grads
from linear_attention_chunks64 import attend_with_grads as expected

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (FP32, 64)])
@pytest.mark.parametrize("bits", [{"v": 50, "S0": 50}, {"do": 40, "dS": 40, "v": 10}, {"v": -40, "S0": -40, "do": -30, "dS": -30}],
                         ids=["large values", "large cotangents", "small"])
@pytest.mark.parametrize("decay", [-0.97, -0.01, "strong"])
def test_large_and_small_numbers(dtype, D, bits, decay):
    """With -0.97 a chunk decays by 2^-90: what its first tokens write is far larger against its end than it is at its end."""
    d = make(1, 200, 1, 2, D, dtype, 41, gate="strong" if decay == "strong" else "token")
    if decay != "strong":
        d["g"].fill_(decay)
    for n, b in bits.items():
        d[n] = d[n] * 2.0 ** b
    check(run_with_grads(d), expected(d), d)


@pytest.mark.parametrize("B,T,HV,D,dtype", [(1, 1, 2, 128, BF16), (1, 3, 2, 64, FP32), (2, 40, 1, 8, FP32), (40, 2, 4, 128, FP32), (75, 1, 2, 64, BF16)])
@pytest.mark.parametrize("g", [0.0, -0.3])
def test_an_infinite_state_stays_infinite(B, T, HV, D, dtype, g):
    """Token by token: a decay multiplies it, and infinity times a decay is infinity.  Nothing else moves."""
    from delta_feedback_experiment_b200 import fused_recurrent_linear_attention as step
    d = make(B, T, 1, HV, D, dtype, 42)
    d["g"].fill_(g)
    d["q"] = d["q"].abs() + 0.01
    clean, S1 = step(*(d[n] for n in NAMES), initial_state=d["S0"], output_final_state=True)
    S0 = d["S0"].clone()
    S0[0, 0, 2, 3], S0[0, 0, 1, 5] = float("inf"), -float("inf")
    o, S = step(*(d[n] for n in NAMES), initial_state=S0, output_final_state=True)
    assert (S[0, 0, 2, 3] == float("inf")) and S[0, 0, 1, 5] == -float("inf")
    assert (o[0, :, 0, 3] == float("inf")).all() and (o[0, :, 0, 5] == -float("inf")).all()
    S[0, 0, 2, 3], S[0, 0, 1, 5] = S1[0, 0, 2, 3], S1[0, 0, 1, 5]
    o[0, :, 0, 3], o[0, :, 0, 5] = clean[0, :, 0, 3], clean[0, :, 0, 5]
    assert torch.equal(S, S1) and torch.equal(o, clean)


@pytest.mark.parametrize("D", [128, 64])
def test_an_infinite_state_in_chunks_stays_with_its_column(D):
    """The state is kept; what reads it takes it in two bf16 parts, whose difference is no number."""
    d = make(1, 150, 1, 2, D, BF16, 43)
    d["g"].fill_(-0.02)
    clean, S1 = attend(d)
    S0 = d["S0"].clone()
    S0[0, 1, 2, 3] = float("inf")
    o, S = attend({**d, "S0": S0})
    assert S[0, 1, 2, 3] == float("inf") and not o[0, :, 1, 3].isfinite().any()
    S[0, 1, 2, 3] = S1[0, 1, 2, 3]
    o[0, :, 1, 3] = clean[0, :, 1, 3]
    assert torch.equal(S, S1) and torch.equal(o, clean)
