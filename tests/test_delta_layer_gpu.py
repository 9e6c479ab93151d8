"""A token mixer out of the operators, as a model runs them: layer norm, projections, the Q|K|V
convolution, the gated delta rule and the norm gate, trained over whole rows (eagerly, under
activation checkpointing, in a captured graph) and then decoded token by token from a prompt's
state.  The whole layer is compared with the same layer in 64 bits."""

import pytest
import torch
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

from conftest import rel_rms
from oracle.delta_rule_oracle import delta_rule_oracle, layer_norm_oracle
from oracle.pkda_layer_oracle import norm_gate_oracle, qkv_conv_oracle

pytestmark = pytest.mark.gpu
bf16, f32 = torch.bfloat16, torch.float32
CUDA = "cuda"

# Root mean squares.  bf16: every rounding is off by at most 2^-8 of its value.  An output lies behind those of the norm, the
# projection, the convolution, the rule's operands and output, and the gate: 8 at most if they lined up; its gradients lie behind
# as many again.  fp32: each operator is within 1e-4 by its own tests; four of them forward, four more backward.
TOL = {bf16: (8 * 2.0 ** -8, 16 * 2.0 ** -8), f32: (4e-4, 8e-4)}


def layer_weights(H, D, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    W = H * D
    n = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    w = {"norm_w": 1 + 0.1 * n(W), "norm_b": 0.1 * n(W), "qkv": n(3 * W, W) * W ** -0.5, "conv": 0.5 * n(3 * W, 4),
         "g": n(H, W) * W ** -0.5, "beta": n(H, W) * W ** -0.5, "gate": n(W, W) * W ** -0.5, "out_norm": 1 + 0.1 * n(D)}
    keep = ("norm_w", "norm_b", "conv", "out_norm")
    return {k: (t if k in keep else t.to(dtype)).to(CUDA) for k, t in w.items()}


def up_to_the_rule(x, w, H, D):
    from delta_feedback_experiment_b200 import layer_norm, pkda_qkv_conv
    B, T, W = x.shape
    y = layer_norm(x, w["norm_w"], w["norm_b"])
    qkv = pkda_qkv_conv(F.linear(y, w["qkv"]), w["conv"], D, 2 * W, 1e-6)
    q, k, v = (t.view(B, T, H, D) for t in qkv)
    return q, k, v, -F.softplus(F.linear(y, w["g"]).float()), torch.sigmoid(F.linear(y, w["beta"])), \
        F.linear(y, w["gate"]).view(B, T, H, D)


def layer(x, w, H, D, state=None):
    from delta_feedback_experiment_b200 import chunk_gated_delta_rule, pkda_norm_gate
    q, k, v, g, beta, gate = up_to_the_rule(x, w, H, D)
    o, S = chunk_gated_delta_rule(q, k, v, g, beta, initial_state=state, output_final_state=True)
    return x + pkda_norm_gate(o, gate, w["out_norm"], 1e-6)[0].reshape(x.shape), S


def layer_oracle(x, w, H, D, state=None):
    B, T, W = x.shape
    y = layer_norm_oracle(x, w["norm_w"], w["norm_b"])
    qkv = qkv_conv_oracle(y @ w["qkv"].T, w["conv"], D, 2 * W, 1e-6, torch.float64)
    q, k, v = (t.reshape(B, T, H, D) for t in qkv)
    g, beta = -F.softplus(y @ w["g"].T), torch.sigmoid(y @ w["beta"].T)
    o, S = delta_rule_oracle(q, k, v, g, beta, None, state)
    gate = (y @ w["gate"].T).reshape(B, T, H, D)
    return x + norm_gate_oracle(o, gate, w["out_norm"], 1e-6, torch.float64)[0].reshape(x.shape), S


def inputs(B, T, H, D, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((B, T, H * D), generator=gen).to(dtype).to(CUDA)
    state = (0.3 * torch.randn((B, H, D, D), generator=gen)).to(CUDA)
    dy = torch.randn((B, T, H * D), generator=gen).to(dtype).to(CUDA)
    dS = (0.3 * torch.randn((B, H, D, D), generator=gen)).to(CUDA)
    return x, state, dy, dS


def grads_of(fn, x, w, state, dy, dS):
    leaves = {"x": x, "state": state, **w}
    leaves = {n: t.detach().clone().requires_grad_(True) for n, t in leaves.items()}
    y, S = fn(leaves["x"], {n: leaves[n] for n in w}, leaves["state"])
    got = torch.autograd.grad([y, S], list(leaves.values()), [dy, dS])
    return {"y": y.detach(), "S": S.detach()}, dict(zip(leaves, got))


@pytest.mark.parametrize("B,T,H,D,dtype", [(2, 130, 2, 128, bf16), (1, 1, 2, 128, bf16), (2, 77, 3, 64, f32)])
def test_layer_matches_the_layer_in_64_bits(B, T, H, D, dtype):
    w = layer_weights(H, D, dtype, seed=1)
    x, state, dy, dS = inputs(B, T, H, D, dtype, seed=2)
    outs, grads = grads_of(lambda a, b, c: layer(a, b, H, D, c), x, w, state, dy, dS)
    up = lambda t: t.detach().cpu().double()  # noqa: E731
    want, wgrads = grads_of(lambda a, b, c: layer_oracle(a, b, H, D, c), up(x), {n: up(t) for n, t in w.items()}, up(state),
                            up(dy), up(dS))
    for name, t in outs.items():
        assert rel_rms(t, want[name]) < TOL[dtype][0], (name, rel_rms(t, want[name]))
    for name, t in grads.items():
        assert t.dtype == (x if name == "x" else state if name == "state" else w[name]).dtype
        assert rel_rms(t, wgrads[name]) < TOL[dtype][1], (name, rel_rms(t, wgrads[name]))


@pytest.mark.parametrize("H,D,dtype", [(2, 128, bf16), (2, 64, f32)])
def test_layer_under_checkpointing_is_the_layer(H, D, dtype):
    w = layer_weights(H, D, dtype, seed=3)
    given = inputs(2, 130, H, D, dtype, seed=4)
    plain = grads_of(lambda a, b, c: layer(a, b, H, D, c), given[0], w, *given[1:])
    again = grads_of(lambda a, b, c: checkpoint(lambda *t: layer(t[0], b, H, D, t[1]), a, c, use_reentrant=False),
                     given[0], w, *given[1:])
    for a, b in zip(plain, again):
        assert [n for n in a if not torch.equal(a[n], b[n])] == []


def test_layer_in_a_captured_step():
    H, D = 2, 128
    w = {n: t.requires_grad_(True) for n, t in layer_weights(H, D, bf16, seed=5).items()}
    x, state, dy, dS = inputs(2, 200, H, D, bf16, seed=6)

    def step():
        y, S = layer(x, w, H, D, state)
        return [y, S, *torch.autograd.grad([y, S], list(w.values()), [dy, dS])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (7, 8):
        for t, new in zip((x, state, dy, dS), inputs(2, 200, H, D, bf16, seed)):
            t.copy_(new)
        graph.replay()
        eager = step()
        assert [i for i, (a, b) in enumerate(zip(captured, eager)) if not torch.equal(a, b)] == []


@pytest.mark.parametrize("H,D,dtype", [(2, 128, bf16), (3, 64, f32)])
def test_decoding_goes_on_from_a_prompt(H, D, dtype):
    """A prompt of 70 tokens by the chunked operator, three tokens at once and eight one by one by the recurrent
    one, the state updated in place: the outputs and the state are the whole row's."""
    from delta_feedback_experiment_b200 import chunk_gated_delta_rule, fused_recurrent_gated_delta_rule, pkda_norm_gate
    B, T, prompt = 2, 81, 70
    w = layer_weights(H, D, dtype, seed=9)
    x, state, _, _ = inputs(B, T, H, D, dtype, seed=10)
    with torch.no_grad():
        q, k, v, g, beta, gate = up_to_the_rule(x, w, H, D)
        cut = lambda a, b: [t[:, a:b] for t in (q, k, v, g, beta)]  # noqa: E731  (strided views: used as they are)
        o, S = chunk_gated_delta_rule(*cut(0, prompt), initial_state=state, output_final_state=True)
        outs = [o]
        ends = [prompt, prompt + 3, *range(prompt + 4, T + 1)]
        for a, b in zip(ends[:-1], ends[1:]):
            o, S2 = fused_recurrent_gated_delta_rule(*cut(a, b), initial_state=S, output_final_state=True, inplace_state=True)
            assert S2.data_ptr() == S.data_ptr()
            outs.append(o)
        y = x + pkda_norm_gate(torch.cat(outs, 1), gate, w["out_norm"], 1e-6)[0].reshape(x.shape)
    up = lambda t: t.detach().cpu().double()  # noqa: E731
    want, want_S = layer_oracle(up(x), {n: up(t) for n, t in w.items()}, H, D, up(state))
    assert rel_rms(y, want) < TOL[dtype][0]
    assert rel_rms(y[:, prompt:], want[:, prompt:]) < TOL[dtype][0]
    assert rel_rms(S, want_S) < TOL[dtype][0]
