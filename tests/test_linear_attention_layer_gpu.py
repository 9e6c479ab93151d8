"""A token mixer out of the operators, as a model runs them: one projection, the norm and rotation of its query and key
slices, linear attention and the norm gate, trained over whole rows (eagerly, under activation checkpointing, in a captured
graph) and then decoded token by token from a prompt's state.  The whole layer is compared with the same layer in 64 bits."""

import functools

import pytest
import torch
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

from conftest import assert_close, rel_rms
from linear_attention_cases import HALF_STEP, SPLIT, make, run_with_grads
from oracle.linear_attention_oracle import attend, norm_rotate
from oracle.pkda_layer_oracle import norm_gate_oracle

pytestmark = pytest.mark.gpu
bf16, f32 = torch.bfloat16, torch.float32

# Root mean squares.  bf16: a rounding is off by at most 2^-8 of its value.  An output lies behind those of the projection, the
# norm and rotation, the attention and the gate: 4 at most if they lined up; its gradients lie behind as many again, and behind the
# weights' own sums.  fp32: each operator is within 1e-4 by its own tests; three forward, three more backward.
TOL = {bf16: (4 * 2.0 ** -8, 9 * 2.0 ** -8), f32: (3e-4, 6e-4)}


def weights(H, HK, D, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    W = H * D
    n = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    w = {"qkv": n((2 * HK + H) * D, W) * W ** -0.5, "gate": n(W, W) * W ** -0.5, "qw": 1 + 0.1 * n(D), "kw": 1 + 0.1 * n(D),
         "decay": -torch.exp2(-torch.arange(1.0, H + 1)), "out": 1 + 0.1 * n(D)}
    return {k: (t.to(dtype) if k in ("qkv", "gate") else t).cuda() for k, t in w.items()}


CPU_FREQ = {D: (10000.0 ** (-torch.arange(0, D, 2) / D)).float() for D in (64, 128)}


@functools.lru_cache
def freq(D, device):
    return CPU_FREQ[D].to(device)


def layer(x, w, H, HK, D, state=None, first=0, step=False):
    from delta_feedback_experiment_b200 import (chunk_linear_attention, fused_recurrent_linear_attention, pkda_norm_gate,
                                                qk_norm_rotate)
    B, T, W = x.shape
    row = F.linear(x, w["qkv"])
    q, k = row[..., :HK * D].unflatten(-1, (HK, D)), row[..., HK * D:2 * HK * D].unflatten(-1, (HK, D))
    v = row[..., 2 * HK * D:].unflatten(-1, (H, D))
    at = torch.arange(first, first + T, device=x.device)
    q, k = qk_norm_rotate(q, k, w["qw"], w["kw"], freq(D, x.device), at)
    run = fused_recurrent_linear_attention if step else chunk_linear_attention
    o, S = run(q, k, v, w["decay"], scale=1.0 / D, initial_state=state, output_final_state=True)
    gate = F.linear(x, w["gate"]).view(B, T, H, D)
    return x + pkda_norm_gate(o, gate, w["out"], 1e-6)[0].reshape(x.shape), S


def definition(x, w, H, HK, D, state=None):
    B, T, W = x.shape
    row = x @ w["qkv"].T
    q, k = row[..., :HK * D].unflatten(-1, (HK, D)), row[..., HK * D:2 * HK * D].unflatten(-1, (HK, D))
    v = row[..., 2 * HK * D:].unflatten(-1, (H, D))
    q, k = (norm_rotate(t, w[n], CPU_FREQ[D]) for t, n in ((q, "qw"), (k, "kw")))
    o, S = attend(q, k, v, w["decay"], 1.0 / D, state)
    gate = (x @ w["gate"].T).reshape(B, T, H, D)
    return x + norm_gate_oracle(o, gate, w["out"], 1e-6, torch.float64)[0].reshape(x.shape), S


def inputs(B, T, H, D, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    return (n(B, T, H * D).to(dtype).cuda(), (0.3 * n(B, H, D, D)).cuda(), n(B, T, H * D).to(dtype).cuda(),
            (0.3 * n(B, H, D, D)).cuda())


def grads_of(fn, x, w, state, dy, dS):
    leaves = {n: t.detach().clone().requires_grad_(True) for n, t in {"x": x, "state": state, **w}.items()}
    y, S = fn(leaves["x"], {n: leaves[n] for n in w}, leaves["state"])
    got = torch.autograd.grad([y, S], list(leaves.values()), [dy, dS])
    return {"y": y.detach(), "S": S.detach()}, dict(zip(leaves, got))


@pytest.mark.parametrize("B,T,H,HK,D,dtype", [(2, 130, 2, 2, 128, bf16), (1, 1, 2, 1, 128, bf16), (2, 77, 4, 2, 64, bf16),
                                              (2, 77, 3, 1, 64, f32)])
def test_trained_eagerly_checkpointed_and_captured(B, T, H, HK, D, dtype):
    x, state, dy, dS = inputs(B, T, H, D, dtype, 1)
    w = weights(H, HK, D, dtype, 2)
    run = lambda x, w, s: layer(x, w, H, HK, D, s)  # noqa: E731
    values, grads = grads_of(run, x, w, state, dy, dS)
    dbl = lambda t: t.detach().double().cpu()  # noqa: E731
    ref, ref_grads = grads_of(lambda x, w, s: definition(x, w, H, HK, D, s), dbl(x), {n: dbl(t) for n, t in w.items()}, dbl(state),
                              dbl(dy), dbl(dS))
    for got, want, tol in ((values, ref, TOL[dtype][0]), (grads, ref_grads, TOL[dtype][1])):
        for n in got:
            assert rel_rms(got[n], want[n]) <= tol, (n, rel_rms(got[n], want[n]))
    again, grads2 = grads_of(lambda x, w, s: checkpoint(run, x, w, s, use_reentrant=False), x, w, state, dy, dS)
    for n in grads:
        assert torch.equal(grads[n], grads2[n]), n

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads_of(run, x, w, state, dy, dS)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, captured = grads_of(run, x, w, state, dy, dS)
    graph.replay()
    assert torch.equal(out["y"], values["y"])
    for n in grads:
        assert torch.equal(captured[n], grads[n]), n


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64)])
def test_decoded_from_a_prompt(dtype, D):
    B, T, H, HK, more = 2, 100, 4, 2, 12
    x, state, _, _ = inputs(B, T + more, H, D, dtype, 3)
    w = weights(H, HK, D, dtype, 4)
    with torch.no_grad():
        whole, S_all = layer(x, w, H, HK, D, state)
        part, S = layer(x[:, :T], w, H, HK, D, state)
        steps = []
        for t in range(T, T + more):
            y, S = layer(x[:, t:t + 1], w, H, HK, D, S, first=t, step=True)
            steps.append(y)
    assert rel_rms(torch.cat([part, *steps], 1), whole.double()) <= 2 * TOL[dtype][0]
    assert rel_rms(S, S_all.double()) <= TOL[dtype][0]


@pytest.mark.parametrize("D", [128, 64])
def test_walked_and_side_by_side_agree(D):
    """Many units are walked from segment to segment by one CTA each, few run their segments side by side: 160 and 2 units of the
    same 1,400 tokens.  Both are off by SPLIT and their rounding at most; the rows of a batch are the same bit for bit."""
    d = make(1, 1400, 1, 2, D, bf16, 5, strength=0.02)
    wide = {n: t if t is None else t.expand(80, *t.shape[1:]).contiguous() for n, t in d.items()}
    few, many = run_with_grads(d), run_with_grads(wide)
    for n, t in many.items():
        assert torch.equal(t, t[:1].expand_as(t)), n
        rtol = 4 * SPLIT if t.dtype == f32 else 2 * SPLIT + 2 * HALF_STEP
        assert_close(t[:1], few[n].double(), rtol, n, outlier_frac=0.0)


def test_two_streams_at_once():
    """Calls on two streams share nothing: the same results as one after the other."""
    a, b = (make(2, 700, 2, 4, 128, bf16, s) for s in (6, 7))
    want = [run_with_grads(t) for t in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, t in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(run_with_grads(t))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for n in g:
                assert torch.equal(g[n], w[n]), n


@pytest.mark.parametrize("D", [128, 64])
def test_a_wait_that_gave_up_marks_the_results(D):
    """With the status word set from the host, as a wait that ran out would leave it, states and first rows are NaN."""
    from delta_feedback_experiment_b200 import _lib, ops
    lib = _lib.load()
    d = make(2, 200, 1, 2, D, bf16, 8)
    clean = run_with_grads(d)
    assert int(ops.last_device_status()) == 0 and int(ops.last_backward_status()) == 0
    assert lib.pkda_set_variant(b"la_chunks", 1) == 0
    try:
        got = run_with_grads(d)
        assert int(ops.last_device_status()) != 0 and int(ops.last_backward_status()) != 0
    finally:
        assert lib.pkda_set_variant(b"la_chunks", 0) == 0
    assert got["S"].isnan().all() and got["dS0"].isnan().all()
    for n in ("o", "dq", "dk", "dv"):
        assert got[n][:, 0].isnan().any(), n
    again = run_with_grads(d)
    for n in clean:
        assert torch.equal(again[n], clean[n]), n


def test_a_gate_that_is_no_number_stays_with_its_head():
    d = make(1, 300, 2, 2, 128, bf16, 9)
    clean = run_with_grads(d)
    d["g"][0, 130, 1] = float("nan")
    got = run_with_grads(d)
    for n in ("o", "dv", "dq", "dk"):
        assert torch.equal(got[n][:, :, 0], clean[n][:, :, 0]), n
    assert torch.equal(got["dg"][..., 0], clean["dg"][..., 0])
    assert torch.equal(got["o"][:, :128, 1], clean["o"][:, :128, 1]) and got["o"][:, 130:, 1].isnan().all()
