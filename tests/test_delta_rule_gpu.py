"""The gated delta rule on the GPU against the token-by-token definition in 64 bits."""

import pytest
import torch

import delta_rule_cases as cases
from conftest import assert_close
from delta_rule_cases import FP32_RTOL, HALF_STEP, check, expected, make, rule, run_with_grads
from oracle.delta_rule_oracle import delta_rule_oracle

pytestmark = pytest.mark.gpu
bf16, f32 = torch.bfloat16, torch.float32
CUDA = "cuda"


def recurrent(d, **kw):
    from delta_feedback_experiment_b200 import fused_recurrent_gated_delta_rule
    return fused_recurrent_gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], initial_state=d["S0"],
                                            output_final_state=True, **kw)


def is_chunked(dtype, D):
    return dtype == bf16 and D == 128


def oracle(d, cu=None):
    f = lambda t: None if t is None else t.cpu().double()  # noqa: E731
    return delta_rule_oracle(*(f(d[n]) for n in ("q", "k", "v", "g", "beta")), None, f(d["S0"]), cu)


def run_output_with_grads(d, cu=None):
    leaves = {n: d[n].detach().clone().requires_grad_(True) for n in ("q", "k", "v", "g", "beta")}
    o, _ = rule({**d, **leaves}, cu=cu, final=False)
    grads = torch.autograd.grad(o, list(leaves.values()), d["do"])
    return {"o": o.detach(), **{"d" + n: t for n, t in zip(leaves, grads)}}


# ------------------------------------------------------------------------- recurrent
@pytest.mark.parametrize("dtype", [bf16, f32])
@pytest.mark.parametrize("B,T,HK,HV,D,state", [
    (1, 1, 1, 1, 8, True), (3, 1, 2, 4, 16, False), (2, 1, 1, 3, 32, True), (2, 1, 2, 2, 64, True),
    (5, 1, 4, 12, 128, True), (2, 2, 2, 4, 128, True), (1, 2, 1, 1, 8, False), (2, 3, 1, 2, 16, True),
    (1, 17, 2, 4, 32, True), (2, 48, 1, 3, 64, True), (1, 65, 2, 2, 128, False), (1, 33, 1, 2, 8, True)])
def test_recurrent_matches_definition(B, T, HK, HV, D, state, dtype):
    d = make(B, T, HK, HV, D, dtype, seed=T + D, state=state)
    o, S = recurrent(d)
    wo, wS = oracle(d)
    assert o.dtype == dtype and S.dtype == f32
    assert_close(o, wo, FP32_RTOL + (HALF_STEP if dtype == bf16 else 0), "o", outlier_frac=0.0)
    assert_close(S, wS, FP32_RTOL, "S")


@pytest.mark.parametrize("T", [1, 2, 5])
def test_recurrent_updates_the_state_in_place(T):
    d = make(3, T, 2, 4, 128, bf16, seed=1)
    o, S = recurrent(d)
    mine = d["S0"].clone()
    o2, S2 = recurrent({**d, "S0": mine}, inplace_state=True)
    assert S2.data_ptr() == mine.data_ptr() and torch.equal(o, o2) and torch.equal(S, mine)


def test_recurrent_steps_follow_one_another():
    """A prompt at once, and token by token through the cached state."""
    d = make(2, 9, 2, 4, 64, f32, seed=2)
    o, S = recurrent(d)
    state, rows = d["S0"].clone(), []
    for t in range(9):
        step = {n: d[n][:, t:t + 1] for n in ("q", "k", "v", "g", "beta")}
        rows.append(recurrent({**step, "S0": state}, inplace_state=True)[0])
    assert_close(torch.cat(rows, 1), o, FP32_RTOL, "o")
    assert_close(state, S, FP32_RTOL, "S")


@pytest.mark.parametrize("B,D,dtype", [(8, 128, f32), (6, 128, f32), (10, 64, f32), (10, 64, bf16), (20, 32, f32)])
def test_many_states(B, D, dtype):
    """Enough (row, head) states that a lane has several of their columns: forward, reverse and the recurrent call."""
    d = make(B, 21, 4, 8, D, dtype, seed=16)
    want = expected(d)
    check(run_with_grads(d), want, False, "chunk")
    o, S = recurrent(d)
    check({"o": o, "S": S}, {n: want[n] for n in ("o", "S")}, False, "recurrent")
    d = make(B, 21, 4, 8, 128, bf16, seed=17)
    o, S = recurrent(d)
    want = oracle(d)
    check({"o": o, "S": S}, {"o": want[0], "S": want[1]}, False, "recurrent, bf16")


# --------------------------------------------------------------------------- chunked
SHAPES = [
    # B, T, HK, HV, D, dtype, state
    (1, 1, 1, 1, 128, bf16, True), (2, 63, 1, 2, 128, bf16, False), (1, 64, 2, 2, 128, bf16, True),
    (2, 65, 1, 3, 128, bf16, True), (3, 130, 2, 4, 128, bf16, False), (1, 517, 1, 2, 128, bf16, True),
    (1, 1, 1, 2, 64, f32, True), (2, 70, 2, 2, 64, f32, True), (1, 200, 1, 3, 128, f32, True),
    (1, 130, 1, 2, 32, f32, False), (2, 33, 1, 1, 16, bf16, True), (1, 97, 2, 4, 8, f32, True),
    (1, 80, 2, 4, 64, bf16, False)]


@pytest.mark.parametrize("strong", [False, True], ids=["mild", "strong"])
@pytest.mark.parametrize("B,T,HK,HV,D,dtype,state", SHAPES)
def test_forward_and_gradients_match_definition(B, T, HK, HV, D, dtype, state, strong):
    d = make(B, T, HK, HV, D, dtype, seed=3 * T + D, state=state, strong=strong)
    got, want = run_with_grads(d), expected(d)
    assert got["dq"].dtype == dtype and got["dg"].dtype == f32 and got["dbeta"].dtype == dtype
    check(got, want, is_chunked(dtype, D), f"{B}x{T}x{HK}/{HV}x{D}")


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64)])
def test_forward_alone_is_the_training_forward(dtype, D):
    d = make(2, 150, 2, 4, D, dtype, seed=5)
    got = run_with_grads(d)
    o, S = rule(d)
    assert torch.equal(o, got["o"]) and torch.equal(S, got["S"])
    o2, none = rule(d, final=False)
    assert none is None and torch.equal(o, o2)


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 32)])
@pytest.mark.parametrize("cu", [[0, 1, 2, 3], [0, 64, 128, 131], [0, 0, 5, 5, 70, 200], [0, 130], [3, 40, 190, 190]],
                         ids=["ones", "whole", "empty", "single", "edges"])
def test_packed_sequences(cu, dtype, D):
    """Lengths of zero and one, whole chunks, rows in front of the first sequence and behind the last."""
    T, N = cu[-1] + 7, len(cu) - 1
    d = make(1, T, 1, 2, D, dtype, seed=T, N=N)
    for n in ("q", "k", "v", "do", "beta"):  # rows that no sequence owns, and nobody reads
        d[n][:, cu[-1]:] = float("nan")
        d[n][:, :cu[0]] = float("nan")
    got = run_with_grads(d, cu=torch.tensor(cu, device=CUDA))
    clean = {k: (torch.nan_to_num(t, nan=0.0) if t is not None else None) for k, t in d.items()}
    want = expected(clean, cu)
    check(got, want, is_chunked(dtype, D), str(cu))
    for n in ("o", "dq", "dk", "dv", "dg", "dbeta"):
        assert (got[n][:, cu[-1]:] == 0).all() and (got[n][:, :cu[0]] == 0).all(), n


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64)])
def test_a_neighbours_nan_stays_with_it(dtype, D):
    """A row of a packed batch or of a batch that holds NaN leaves the others as they are."""
    d = make(1, 150, 1, 2, D, dtype, seed=8, N=2)
    cu = torch.tensor([0, 70, 150], device=CUDA)
    clean = run_with_grads(d, cu=cu)
    d["v"][0, 75], d["k"][0, 80] = float("nan"), float("inf")
    d["do"][0, 71] = float("nan")
    got = run_with_grads(d, cu=cu)
    for n in ("o", "dq", "dk", "dv", "dg", "dbeta"):
        assert torch.equal(got[n][:, :70], clean[n][:, :70]), n
    assert torch.equal(got["S"][0], clean["S"][0]) and torch.equal(got["dS0"][0], clean["dS0"][0])
    assert not torch.isfinite(got["o"][0, 75:]).all()


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64), (bf16, 16)])
def test_forgetting_everything(dtype, D):
    """g = -inf at a token: nothing before it reaches anything after, gradients stay finite."""
    d = make(1, 140, 1, 2, D, dtype, seed=9)
    d["g"][0, 0, 0] = d["g"][0, 37] = d["g"][0, 64, 1] = d["g"][0, 128] = float("-inf")
    d["g"][0, 100] = torch.finfo(f32).min
    want = expected({**d, "g": d["g"].clamp(min=-1000.0)})
    check(run_with_grads(d), want, is_chunked(dtype, D), "reset")
    o, S = recurrent(d)
    assert_close(o, want["o"], FP32_RTOL + (HALF_STEP if dtype == bf16 else 0), "o", outlier_frac=0.0)


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64)])
def test_tokens_that_write_nothing(dtype, D):
    """beta = 0 (a masked token), zero keys, beta = 1 with equal keys (the write replaces what was there), no decay."""
    d = make(2, 100, 1, 2, D, dtype, seed=10)
    d["beta"][0, 10:80] = 0
    d["k"][1, 5:20] = 0
    d["k"][1, 40:70] = d["k"][1, 40:41].clone()
    d["beta"][1, 40:70] = 1
    d["g"][:, 30:] = 0
    check(run_with_grads(d), expected(d), is_chunked(dtype, D), "masked")


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64)])
def test_strides_alignments_and_types(dtype, D):
    B, T, HK, HV = 2, 70, 2, 4
    d = make(B, T, HK, HV, D, dtype, seed=11)
    want = run_with_grads(d)
    odd = dict(d)
    odd["q"] = d["q"].transpose(1, 2).contiguous().transpose(1, 2)                # other strides
    wide = torch.zeros(B, T, HK * D + HV * D, device=CUDA, dtype=dtype)
    wide[..., HK * D:] = d["v"].reshape(B, T, -1)
    odd["v"] = wide[..., HK * D:].unflatten(-1, (HV, D))                          # a slice of a packed projection
    flat = torch.zeros(d["k"].numel() + 1, device=CUDA, dtype=dtype)
    flat[1:] = d["k"].flatten()
    odd["k"] = flat[1:].view_as(d["k"])                                           # off the 16-byte grid
    odd["do"] = d["do"].flip(1).contiguous().flip(1)
    odd["S0"] = d["S0"].transpose(0, 1).contiguous().transpose(0, 1)
    state = torch.zeros(d["dS"].numel() + 3, device=CUDA)
    state[3:] = d["dS"].flatten()
    odd["dS"] = state[3:].view_as(d["dS"])
    got = run_with_grads(odd)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    expanded = {**d, "v": d["v"][:1].expand(B, T, HV, D)}                          # a broadcast value
    same = {**d, "v": d["v"][:1].expand(B, T, HV, D).contiguous()}
    a, b = run_with_grads(expanded), run_with_grads(same)
    assert all(torch.equal(a[n], b[n]) for n in a)
    # other types of the scalars are converted, their gradients come back in them
    low = {**d, "g": d["g"].to(bf16), "beta": d["beta"].double()}
    got = run_with_grads(low)
    assert got["dg"].dtype == bf16 and got["dbeta"].dtype == torch.float64


def test_one_tensor_in_two_places():
    """q and k as one and the same leaf: its gradient is the sum of both."""
    d = make(1, 90, 2, 2, 128, bf16, seed=12)
    x = d["k"].clone().requires_grad_(True)
    o, _ = rule({**d, "q": x, "k": x})
    (dx,) = torch.autograd.grad(o, x, d["do"])
    two = run_with_grads({**d, "q": d["k"], "dS": None})
    assert torch.equal(dx, two["dq"] + two["dk"])


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64)])
def test_only_the_final_state_has_a_cotangent(dtype, D):
    d = make(1, 100, 1, 2, D, dtype, seed=13)
    leaves = {n: d[n].clone().requires_grad_(True) for n in ("q", "k", "v", "g", "beta", "S0")}
    _, S = rule({**d, **leaves})
    got = torch.autograd.grad(S, list(leaves.values()), d["dS"])
    want = expected({**d, "do": torch.zeros_like(d["do"])})
    assert (got[0] == 0).all()
    check({"d" + n: t for n, t in zip(leaves, got) if n != "q"},
          {"d" + n: want["d" + n] for n in leaves if n != "q"}, is_chunked(dtype, D), "state only")


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64)])
def test_calls_repeat_bit_for_bit(dtype, D):
    d = make(2, 333, 2, 6, D, dtype, seed=14)
    a, b = run_with_grads(d), run_with_grads(d)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("B,T,HK,HV", [(2, 333, 2, 6), (1, 1000, 2, 8), (3, 777, 1, 5), (2, 320, 6, 6)])
def test_many_calls_repeat(B, T, HK, HV):
    """Small calls whose tiles come from L2, as fast as tiles come: what one head's warps still read must not be
    overwritten by the next head's."""
    d = make(B, T, HK, HV, 128, bf16, seed=14)
    first = run_with_grads(d)
    for _ in range(300):
        got = run_with_grads(d)
        assert [n for n in first if not torch.equal(first[n], got[n])] == []


@pytest.mark.parametrize("B,T,HK,HV,state", [(1, 1025, 1, 2, True), (2, 1500, 2, 6, False), (1, 4096, 4, 4, True),
                                             (3, 2047, 3, 24, True), (1, 1025, 74, 74, False), (1, 2118, 10, 10, True),
                                             (2, 2200, 8, 16, False)])
def test_long_rows_of_few_heads(B, T, HK, HV, state):
    """Such a dense call is taken in two parts, a packed one is not: the same numbers, and so in a replayed graph and from call to
    call."""
    d = make(B, T, HK, HV, 128, bf16, seed=18, state=state)
    got = run_with_grads(d) if state else run_output_with_grads(d)
    flat = {n: t if t is None or n in ("S0", "dS") else t.reshape(1, B * T, *t.shape[2:]) for n, t in d.items()}
    cu = torch.arange(B + 1, dtype=torch.int32, device=CUDA) * T
    want = run_with_grads(flat, cu) if state else run_output_with_grads(flat, cu)
    assert [n for n in got if not torch.equal(got[n].reshape(want[n].shape), want[n])] == []
    for _ in range(20):
        again = run_with_grads(d) if state else run_output_with_grads(d)
        assert [n for n in got if not torch.equal(got[n], again[n])] == []
    with torch.no_grad():
        rule(d)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, S = rule(d)
        graph.replay()
        assert torch.equal(o, got["o"]) and (not state or torch.equal(S, got["S"]))


def test_long_rows_replayed_on_new_inputs():
    """Both kinds of launch that run beside another read what the replay before was not given yet."""
    inputs = [make(2, 2200, 8, 16, 128, bf16, seed=s) for s in (30, 31, 32)]
    want = [run_with_grads(d) for d in inputs]
    held = {n: t.clone().requires_grad_(n not in ("do", "dS")) for n, t in inputs[0].items()}

    def step():
        o, S = rule(held)
        return [o, S, *torch.autograd.grad([o, S], [held[n] for n in ("q", "k", "v", "g", "beta", "S0")],
                                           [held["do"], held["dS"]])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(30):
        with torch.no_grad():
            for n in held:
                held[n].copy_(inputs[turn % 3][n])
        graph.replay()
        for n, t in zip(("o", "S", "dq", "dk", "dv", "dg", "dbeta", "dS0"), out):
            assert torch.equal(t, want[turn % 3][n]), (turn, n)


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64)])
def test_gradient_against_differences(dtype, D):
    """Along a random direction of the gates and of the initial state, which fp32 resolves in both paths."""
    d = make(1, 96, 1, 2, D, dtype, seed=15)
    got = run_with_grads(d)
    gen = torch.Generator().manual_seed(0)
    f = lambda e: sum((x.cpu().double() * c.cpu().double()).sum() for x, c in  # noqa: E731
                      zip(oracle(e), (d["do"], d["dS"])))
    for n, step in (("g", 1e-4), ("S0", 1e-3)):
        move = torch.randn(d[n].shape, generator=gen).to(CUDA)
        slope = (f({**d, n: d[n].double() + step * move}) - f({**d, n: d[n].double() - step * move})) / (2 * step)
        mine = (got["d" + n].double() * move).sum().cpu()
        # the slope sums products with both signs: bounded against the norms of its factors
        bound = (cases.BF16_RTOL if is_chunked(dtype, D) else FP32_RTOL) * float(got["d" + n].norm()) * 3
        assert abs(float(slope - mine)) < bound + 1e-5 * abs(float(slope)), n


# ------------------------------------------------------------- streams, graphs, devices
@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64)])
def test_captured_step_replays_on_new_inputs(dtype, D):
    first, second = (make(2, 130, 1, 2, D, dtype, seed=s) for s in (20, 21))
    want = run_with_grads(second)
    held = {n: t.clone().requires_grad_(n not in ("do", "dS")) for n, t in first.items()}

    def step():
        o, S = rule(held)
        return [o, S, *torch.autograd.grad([o, S], [held[n] for n in ("q", "k", "v", "g", "beta", "S0")],
                                           [held["do"], held["dS"]])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        for n in held:
            held[n].copy_(second[n])
    graph.replay()
    torch.cuda.synchronize()
    for n, t in zip(("o", "S", "dq", "dk", "dv", "dg", "dbeta", "dS0"), out):
        assert torch.equal(t, want[n]), n


def test_two_captured_graphs_in_turn():
    """Each graph has scratch of its own: replays in any order give what an eager call gives."""
    runs = []
    for seed, T in ((22, 200), (23, 97)):
        d = make(1, T, 1, 2, 128, bf16, seed=seed)
        want = rule(d)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = rule(d)
        runs.append((graph, got, want, d))  # (the inputs live as long as the graph that reads them)
    for i in (0, 1, 1, 0):
        runs[i][0].replay()
    torch.cuda.synchronize()
    for _, got, want, _ in runs:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_other_stream_and_calls_side_by_side():
    ds = [make(1, 300, 2, 4, 128, bf16, seed=24 + i) for i in range(2)]
    want = [run_with_grads(d) for d in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    torch.cuda.synchronize()
    got = []
    for s, d in zip(streams, ds):
        with torch.cuda.stream(s):
            got.append(run_with_grads(d))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(a[n], b[n]) for n in b)


def test_status_words_stay_clean():
    from delta_feedback_experiment_b200 import ops
    run_with_grads(make(2, 200, 2, 4, 128, bf16, seed=26))
    assert ops.last_device_status() == 0 and ops.last_backward_status() == 0


def test_empty_calls():
    for dtype, D in ((bf16, 128), (f32, 64)):
        d = make(2, 0, 1, 2, D, dtype, seed=27)
        got = run_with_grads(d)
        assert got["o"].shape == (2, 0, 2, D) and torch.equal(got["S"], d["S0"]) and torch.equal(got["dS0"], d["dS"])
        d = make(0, 5, 1, 2, D, dtype, seed=28, state=False)
        o, S = rule(d)
        assert o.shape == (0, 5, 2, D) and S.shape == (0, 2, D, D)
        o, S = recurrent(make(1, 0, 1, 2, D, dtype, seed=29))
        assert o.shape == (1, 0, 2, D)


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64)])
def test_packed_rows_of_no_sequence_at_all(dtype, D):
    d = make(1, 70, 1, 2, D, dtype, seed=19, N=0)
    cu = torch.zeros(1, dtype=torch.int32, device=CUDA)
    junk = torch.full((4 << 20,), float("nan"), device=CUDA)  # (what the allocator hands out next)
    del junk
    got = run_with_grads(d, cu)
    assert got["S"].shape == got["dS0"].shape == (0, 2, D, D)
    assert all((t == 0).all() for t in got.values())
    o, S = recurrent(d, cu_seqlens=cu)
    assert (o == 0).all() and S.shape == (0, 2, D, D)


def test_a_state_updated_in_place_is_a_changed_state():
    d = make(1, 1, 1, 2, 64, f32, seed=20)
    before = d["S0"]._version
    recurrent(d, inplace_state=True)
    assert d["S0"]._version > before
    with pytest.raises(RuntimeError, match="requires grad"):
        recurrent({**d, "S0": d["S0"].clone().requires_grad_(True)}, inplace_state=True)
    with torch.inference_mode():
        recurrent({**d, "S0": d["S0"].clone()}, inplace_state=True)


def test_second_derivatives_are_refused():
    d = make(1, 20, 1, 1, 64, f32, seed=30)
    g = d["g"].clone().requires_grad_(True)
    o, _ = rule({**d, "g": g})
    (dg,) = torch.autograd.grad(o.sum(), g, create_graph=True)
    assert not dg.requires_grad


# ------------------------------------------------------------------------- refusals
def test_wrong_arguments_are_refused_before_any_launch():
    from delta_feedback_experiment_b200 import chunk_gated_delta_rule, fused_recurrent_gated_delta_rule, ops
    d = make(2, 10, 2, 4, 64, f32, seed=31)
    args = [d[n] for n in ("q", "k", "v", "g", "beta")]
    count = ops.LAUNCHES

    def refused(match, changed, **kw):
        a = [changed.get(i, t) for i, t in enumerate(args)]
        for f in (chunk_gated_delta_rule, fused_recurrent_gated_delta_rule):
            with pytest.raises(RuntimeError, match=match):
                f(*a, **kw)
    refused("k has shape", {1: d["k"][:, :9]})
    refused("v has shape", {2: d["v"][..., :32]})
    refused("do not divide", {2: d["v"][:, :, :3]})
    refused("g has shape", {3: d["g"][:, :, :3]})
    refused("k is", {1: d["k"].to(bf16)})
    refused("bf16 or fp32", {0: d["q"].half(), 1: d["k"].half(), 2: d["v"].half()})
    refused("unsupported geometry", {i: d[n][..., :48] for i, n in enumerate("qkv")})
    refused("initial_state has shape", {}, initial_state=d["S0"][:1])
    refused("batch size 1", {}, cu_seqlens=torch.tensor([0, 10], device=CUDA))
    refused("offsets", {i: t[:1] for i, t in enumerate(args)}, cu_seqlens=torch.tensor([0.0, 10.0], device=CUDA))
    refused("different devices|no CPU path", {1: d["k"].cpu()})
    refused("expected q, k|expected, got q", {0: d["q"][0]})
    with pytest.raises(RuntimeError, match="in-place"):
        fused_recurrent_gated_delta_rule(*args, inplace_state=True)
    with pytest.raises(RuntimeError, match="in-place"):
        fused_recurrent_gated_delta_rule(*args, initial_state=d["S0"].to(bf16), inplace_state=True)
    assert ops.LAUNCHES == count


@pytest.mark.parametrize("dtype,D", [(bf16, 128), (f32, 64)])
def test_offsets_out_of_order_stay_inside(dtype, D):
    """What the offsets hold is only known on the device: sequences are cut to the rows there are."""
    d = make(1, 100, 1, 2, D, dtype, seed=32, N=3)
    got = run_with_grads(d, cu=torch.tensor([0, 80, 60, 5000], device=CUDA))
    want = expected(d, [0, 80, 80, 100])
    check(got, want, is_chunked(dtype, D), "cut")
