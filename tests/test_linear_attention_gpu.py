"""chunk_linear_attention and fused_recurrent_linear_attention against the recurrence in 64 bits."""

import pytest
import torch

from conftest import assert_close
from linear_attention_cases import FP32_RTOL, HALF_STEP, NAMES, SPLIT, attend, check, expected, make, run_with_grads

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


def recurrent(d, **kw):
    from delta_feedback_experiment_b200 import fused_recurrent_linear_attention
    return fused_recurrent_linear_attention(*(d[n] for n in NAMES), output_final_state=True, **kw)


@pytest.mark.parametrize("B,T,HK,HV,D,dtype", [
    (1, 1, 1, 1, 8, FP32), (2, 17, 1, 3, 8, FP32), (1, 40, 2, 2, 16, BF16), (2, 33, 2, 4, 16, FP32), (3, 70, 1, 1, 32, BF16),
    (2, 100, 2, 4, 32, FP32), (2, 65, 4, 4, 64, FP32), (1, 130, 2, 6, 128, FP32), (2, 1, 1, 2, 128, FP32)])
@pytest.mark.parametrize("gate", ["token", "head", "strong"])
def test_exact_kernels(B, T, HK, HV, D, dtype, gate):
    d = make(B, T, HK, HV, D, dtype, 1, gate=gate)
    check(run_with_grads(d), expected(d), d)


@pytest.mark.parametrize("B,T,HK,HV,D", [
    (1, 1, 1, 1, 128), (2, 2, 1, 2, 128), (1, 63, 2, 2, 128), (2, 64, 1, 1, 128), (1, 65, 2, 4, 128), (3, 128, 1, 3, 128),
    (1, 333, 2, 2, 128), (2, 200, 3, 3, 128), (1, 1, 2, 2, 64), (2, 64, 1, 2, 64), (1, 65, 2, 2, 64), (2, 257, 2, 6, 64)])
@pytest.mark.parametrize("gate,state", [("token", True), ("head", True), ("strong", False), ("token", False)])
def test_chunked_kernels(B, T, HK, HV, D, gate, state):
    d = make(B, T, HK, HV, D, BF16, 2, gate=gate, state=state)
    check(run_with_grads(d), expected(d), d)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (FP32, 64), (BF16, 32)])
def test_long_rows_cross_segments(dtype, D):
    """More tokens than one segment of a sequence has, weak decay: states have to pass from segment to segment."""
    d = make(1, 1400, 1, 2, D, dtype, 3, strength=0.003)
    check(run_with_grads(d), expected(d), d)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (FP32, 32), (BF16, 16)])
@pytest.mark.parametrize("gate", ["token", "head"])
def test_packed(dtype, D, gate):
    """Sequences of 0, 1, 64, 65 and more tokens, rows in front of the first and behind the last."""
    ends = [3, 3, 4, 68, 133, 133, 300]
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    d = make(1, 311, 2, 4, D, dtype, 4, N=len(ends) - 1, gate=gate)
    for n in ("q", "k", "v", "do"):  # rows that no sequence owns hold anything
        d[n][:, :3] = float("nan")
        d[n][:, 300:] = float("nan")
    got = run_with_grads(d, cu=cu)
    for n in ("o", "dq", "dk", "dv") + (("dg",) if gate == "token" else ()):
        assert not got[n][:, :3].any() and not got[n][:, 300:].any(), n
    for n in ("q", "k", "v", "do"):
        d[n][:, :3] = 0
        d[n][:, 300:] = 0
    check(got, expected(d, cu=ends), d, ends)


def test_many_short_sequences():
    lens = [1 + (7 * i) % 90 for i in range(150)]
    ends = [0]
    for x in lens:
        ends.append(ends[-1] + x)
    cu = torch.tensor(ends, dtype=torch.int64, device="cuda")
    for dtype, D in ((BF16, 128), (FP32, 8)):
        d = make(1, ends[-1], 1, 1, D, dtype, 5, N=len(lens), strength=0.1)
        check(run_with_grads(d, cu=cu), expected(d, cu=ends), d, ends)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP32, 64)])
def test_offsets_that_run_backwards_are_cut(dtype, D):
    """Whatever the offsets say, no row has two owners and nothing outside of the tensors is touched."""
    bad = torch.tensor([0, 100, 50, 400, 160], dtype=torch.int32, device="cuda")
    good = torch.tensor([0, 100, 100, 160, 160], dtype=torch.int32, device="cuda")
    d = make(1, 160, 1, 2, D, dtype, 6, N=4)
    a, b = run_with_grads(d, cu=bad), run_with_grads(d, cu=good)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    from delta_feedback_experiment_b200 import fused_recurrent_linear_attention as step
    x, y = (step(*(d[n] for n in NAMES), initial_state=d["S0"], output_final_state=True, cu_seqlens=c) for c in (bad, good))
    assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (FP32, 64), (BF16, 8)])
def test_a_gate_of_minus_infinity_forgets(dtype, D):
    """-inf at a document's first token equals a new sequence; gates of -200 act like it."""
    d = make(1, 150, 2, 2, D, dtype, 7, state=False)
    d["g"][:, 70] = -float("inf")
    d["g"][:, 131, 0] = -200.0
    got = run_with_grads(d)
    e = {**d, "g": d["g"].clamp_min(-1000.0)}
    want = expected(e)
    want["dg"][:, 70] = 0
    check(got, want, e)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP32, 64)])
def test_without_decay_and_large_scale(dtype, D):
    d = make(2, 130, 1, 2, D, dtype, 8)
    d["g"].zero_()
    check(run_with_grads(d, scale=3.0), expected(d, scale=3.0), d)


@pytest.mark.parametrize("B,T,HK,HV,D,dtype", [(5, 1, 2, 4, 128, BF16), (2, 7, 1, 1, 128, FP32), (2, 48, 2, 2, 64, BF16),
                                               (1, 64, 1, 2, 8, FP32), (300, 1, 1, 1, 128, BF16), (3, 0, 1, 2, 64, FP32)])
def test_recurrent(B, T, HK, HV, D, dtype):
    d = make(B, T, HK, HV, D, dtype, 9)
    o, S = recurrent(d, initial_state=d["S0"])
    want = expected(d) if T else {"o": d["v"].double(), "S": d["S0"].double()}
    if T:
        assert_close(o, want["o"], FP32_RTOL + (HALF_STEP if dtype == BF16 else 0), "o")
    assert_close(S, want["S"], FP32_RTOL, "S")
    state = d["S0"].clone()
    o2, S2 = recurrent({**d, "S0": state}, initial_state=state, inplace_state=True)
    assert S2.data_ptr() == state.data_ptr() and torch.equal(S2, S) and torch.equal(o2, o)


@pytest.mark.parametrize("B,T,HK,HV,D,dtype", [(40, 1, 2, 4, 128, BF16), (37, 2, 2, 4, 128, FP32), (75, 2, 1, 2, 64, BF16), (160, 1, 1, 1, 64, FP32)])
@pytest.mark.parametrize("gate", ["token", "head"])
def test_a_step_of_heads_that_fill_the_device(B, T, HK, HV, D, dtype, gate):
    d = make(B, T, HK, HV, D, dtype, 19, gate=gate)
    d["g"] = d["g"].clone()
    d["g"].view(-1)[0] = float("-inf")
    tol = FP32_RTOL + (HALF_STEP if dtype == BF16 else 0)
    state = d["S0"].clone()
    o, S = recurrent(d, initial_state=state, inplace_state=True)
    want = expected(d)
    assert S.data_ptr() == state.data_ptr()
    assert_close(o, want["o"], tol, "o")
    assert_close(S, want["S"], FP32_RTOL, "S")
    want = expected({**d, "S0": None})
    o, S = recurrent(d)
    assert_close(o, want["o"], tol, "o")
    assert_close(S, want["S"], FP32_RTOL, "S")
    bad = {**d, "g": d["g"].clone()}
    bad["g"].view(-1)[-1] = float("nan")  # the last head's, of the last row or of all
    o2, S2 = recurrent(bad)
    assert S2[-1, -1].isnan().all() and torch.equal(S2[:, :-1], S[:, :-1]) and torch.equal(o2[..., :-1, :], o[..., :-1, :])


def test_recurrent_takes_packed_rows_and_no_state():
    ends = [2, 2, 3, 40, 41]
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    d = make(1, 45, 2, 4, 64, FP32, 10, N=4, gate="head", state=False)
    o, S = recurrent(d, cu_seqlens=cu)
    want = expected(d, cu=ends)
    assert_close(o, want["o"], FP32_RTOL, "o")
    assert_close(S, want["S"], FP32_RTOL, "S")


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (FP32, 64)])
def test_a_prompt_and_steps_equal_one_call(dtype, D):
    d = make(2, 140, 2, 4, D, dtype, 11)
    o, S = attend(d)
    part = {n: d[n][:, :100] for n in NAMES}
    o1, S1 = attend({**part, "S0": d["S0"]})
    steps = []
    for t in range(100, 140):
        o2, S1 = recurrent({n: d[n][:, t:t + 1] for n in NAMES}, initial_state=S1)
        steps.append(o2)
    rtol = 2 * (FP32_RTOL if dtype == FP32 else SPLIT)  # (both sides are off by it)
    assert_close(S1, S, rtol, "S")
    assert_close(torch.cat([o1, *steps], 1), o.double(), rtol + (2 * HALF_STEP if dtype == BF16 else 0), "o")


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP32, 32)])
def test_strided_and_misaligned_inputs(dtype, D):
    d = make(2, 70, 2, 2, D, dtype, 12)
    row = torch.zeros(2, 70, 3 * 2 * D + 3, dtype=dtype, device="cuda")
    v = {}
    for i, n in enumerate(("q", "k", "v")):
        s = row[..., 3 + 2 * i * D:3 + 2 * (i + 1) * D].unflatten(-1, (2, D))
        s.copy_(d[n])
        v[n] = s
    v["g"] = d["g"].transpose(1, 2).contiguous().transpose(1, 2)
    v["S0"] = d["S0"].transpose(-1, -2).contiguous().transpose(-1, -2)
    a, b = attend(d), attend(v)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (FP32, 64)])
def test_gradients_are_deterministic_and_agree_with_differences(dtype, D):
    d = make(2, 200, 2, 4, D, dtype, 13)
    a, b = run_with_grads(d), run_with_grads(d)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    # the loss along one direction, by differences of the 64-bit definition, against the kernels' gradients
    from oracle.linear_attention_oracle import attend as define
    gen = torch.Generator().manual_seed(14)
    x = {n: d[n].double().cpu() for n in (*NAMES, "S0")}
    for n in x:
        direction = torch.randn(x[n].shape, generator=gen, dtype=torch.float64)
        h = 1e-5

        def loss(s):
            y = {**x, n: x[n] + s * h * direction}
            o, S = define(*(y[m] for m in NAMES), None, y["S0"])
            return float((o * d["do"].double().cpu()).sum() + (S * d["dS"].double().cpu()).sum())

        want = (loss(1) - loss(-1)) / (2 * h)
        g = a["d" + n].double().cpu()
        # rounding of the gradient's entries adds up like a random walk: a few times its size times sqrt(entries)
        step = (HALF_STEP if g.dtype == BF16 or (dtype == BF16 and n in "qkv") else 0) + (SPLIT if dtype == BF16 else FP32_RTOL)
        assert abs(float((g * direction).sum()) - want) < 6 * step * float((g * direction).norm()) + 1e-6 * abs(want), n


def test_a_fixed_decay_costs_no_gradient():
    """Without the gate's gradient the same results, in another order of the sums: both are off by half a step of bf16 at most."""
    d = make(1, 90, 1, 2, 128, BF16, 15, gate="head")
    full = run_with_grads(d)
    leaves = {n: d[n].detach().clone().requires_grad_(True) for n in ("q", "k", "v", "S0")}
    o, S = attend({**d, **leaves})
    grads = torch.autograd.grad([o, S], list(leaves.values()), [d["do"], d["dS"]])
    for n, t in zip(leaves, grads):
        assert_close(t, full["d" + n].double(), 2 * SPLIT + (2 * HALF_STEP if t.dtype == BF16 else 0), n, outlier_frac=0.0)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP32, 64)])
def test_nothing_to_do(dtype, D):
    d = make(2, 0, 1, 2, D, dtype, 16)
    got = run_with_grads(d)
    assert torch.equal(got["S"], d["S0"]) and torch.equal(got["dS0"], d["dS"])
    d = make(2, 0, 1, 2, D, dtype, 16, gate="head")
    assert not run_with_grads(d)["dg"].any()
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    d = make(1, 5, 1, 2, D, dtype, 17, N=0, gate="head")
    got = run_with_grads(d, cu=cu)
    assert not any(got[n].any() for n in ("o", "dq", "dk", "dv", "dg"))


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP32, 64)])
def test_captured_training_step_on_another_stream(dtype, D):
    d = make(2, 150, 2, 4, D, dtype, 18)
    leaves = {n: d[n].detach().clone().requires_grad_(True) for n in (*NAMES, "S0")}

    def step():
        o, S = attend({**d, **leaves})
        return [o, S, *torch.autograd.grad([o, S], list(leaves.values()), [d["do"], d["dS"]])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    e = make(2, 150, 2, 4, D, dtype, 19)
    with torch.no_grad():
        for n in leaves:
            leaves[n].copy_(e[n])
        d["do"].copy_(e["do"])
        d["dS"].copy_(e["dS"])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    want = run_with_grads(e)
    for t, n in zip(out, ("o", "S", "dq", "dk", "dv", "dg", "dS0")):
        assert torch.equal(t, want[n]), n


def test_nan_stays_with_its_sequence_and_heads():
    ends = [0, 100, 230]
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    for dtype, D in ((BF16, 128), (BF16, 64), (FP32, 64)):
        d = make(1, 230, 2, 2, D, dtype, 20, N=2)
        clean = run_with_grads(d, cu=cu)
        d["v"][0, 50, 1, 3] = float("nan")
        got = run_with_grads(d, cu=cu)
        assert got["o"][0, 50, 1].isnan().any()
        for n in ("o", "dq", "dk", "dv"):
            assert torch.equal(got[n][:, 100:], clean[n][:, 100:]), n
            assert torch.equal(got[n][:, :, 0], clean[n][:, :, 0]), n


def test_second_derivative_warns_and_recurrent_has_no_gradient():
    d = make(1, 10, 1, 1, 64, FP32, 21)
    q = d["q"].clone().requires_grad_(True)
    o, _ = attend({**d, "q": q})
    with pytest.warns(UserWarning, match="differentiable once"):
        torch.autograd.grad(o.sum(), q, create_graph=True)
    o, S = recurrent({**d, "q": q}, initial_state=d["S0"])
    assert not o.requires_grad and not S.requires_grad


def test_refusals():
    d = make(2, 6, 2, 4, 64, FP32, 22)

    def refuse(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            attend({**d, **kw})
        with pytest.raises(RuntimeError, match=match):
            recurrent({**d, **kw}, initial_state={**d, **kw}["S0"])

    refuse("q has shape|expected q|k has shape", k=d["k"][:, :5])
    refuse("do not divide", v=d["v"][:, :, :3], g=d["g"][:, :, :3])
    refuse("g has shape", g=d["g"][:, :, :3])
    refuse("g has shape", g=d["g"][0, 0, :3])
    refuse("initial_state has shape", S0=d["S0"][:1])
    refuse("is .*BFloat16|is c10::BFloat16", v=d["v"].bfloat16())
    refuse("bf16 or fp32", q=d["q"].half(), k=d["k"].half(), v=d["v"].half())
    refuse("no CPU path", v=d["v"].cpu())
    refuse("floating", g=d["g"].long())
    with pytest.raises(RuntimeError, match="geometry"):
        attend({n: (t[..., :48] if n in "qkv" else None if n == "S0" else t) for n, t in d.items()})
    with pytest.raises(RuntimeError, match="batch size 1"):
        attend(d, cu=torch.tensor([0, 6], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="in-place decode"):
        recurrent(d, initial_state=d["S0"].transpose(-1, -2), inplace_state=True)
    with pytest.raises(RuntimeError, match="requires grad"):
        recurrent(d, initial_state=d["S0"].clone().requires_grad_(True), inplace_state=True)
