"""The decay of a token, formed from its gate in two parts."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_exponential_of_a_gate():
    """A state of ones decayed once: half a step of fp32 for the result, and what the two parts of the decay are off by: a rest of
    at most 2^-5 ln 2 in which six roundings of half a step leave 3 * 2^-24 * 0.022 < 2^-27."""
    from delta_feedback_experiment_b200 import fused_recurrent_linear_attention
    N, H, D = 4096, 64, 8
    gen = torch.Generator().manual_seed(54)
    g = -torch.rand(N, 1, H, generator=gen) * 86
    g[:1024] = -(2.0 ** -(24 * torch.rand(1024, 1, H, generator=gen)))
    g = g.cuda()
    zero = torch.zeros(N, 1, 1, D, device="cuda")
    S0 = torch.ones(N, H, D, D, device="cuda")
    _, S = fused_recurrent_linear_attention(zero, zero, zero.expand(N, 1, H, D), g, initial_state=S0, output_final_state=True)
    want = g[:, 0].double().exp()
    assert torch.equal(S, S[:, :, :1, :1].expand_as(S))
    half = torch.exp2(want.log2().floor() - 24)
    assert ((S[:, :, 0, 0].double() - want).abs() <= half + 2.0 ** -27 * want).all()
