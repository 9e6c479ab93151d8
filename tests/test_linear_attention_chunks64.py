"""The chunked 64-bit form that long rows are compared with is the oracle's token by token."""

import pytest
import torch

import linear_attention_chunks64 as chunks64
from linear_attention_cases import make
from oracle.linear_attention_oracle import attend_with_grads


@pytest.mark.parametrize("gate", ["token", "head", "strong"])
@pytest.mark.parametrize("cu,N,B,T", [(None, 2, 2, 150), ([3, 3, 4, 70, 199], 4, 1, 205)])
def test_same_as_token_by_token(gate, cu, N, B, T):
    d = make(B, T, 1, 2, 8, torch.float32, 1, N=N, gate=gate, device="cpu")
    got, want = chunks64.attend_with_grads(d, cu, 0.7), attend_with_grads(d, cu, 0.7)
    assert set(got) == set(want)
    for n, t in got.items():
        # some hundred roundings of 2^-53, in exponents of up to 2^10 too
        assert (t - want[n]).abs().max() <= 2.0 ** -36 * (1 + want[n].abs().max()), n
