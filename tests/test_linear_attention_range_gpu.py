"""The range of numbers that linear attention takes."""

import pytest
import torch

from linear_attention_cases import check, make, run_with_grads
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
