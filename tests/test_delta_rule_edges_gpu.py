"""The gated delta rule at calls that its documentation allows and that few make."""

import pytest
import torch

from conftest import assert_close
from delta_rule_cases import FP32_RTOL, HALF_STEP, make, rule, run_with_grads
from oracle.delta_rule_oracle import delta_rule_oracle

pytestmark = pytest.mark.gpu
bf16, f32 = torch.bfloat16, torch.float32
CUDA = "cuda"


def recurrent(d, **kw):
    from delta_feedback_experiment_b200 import fused_recurrent_gated_delta_rule
    return fused_recurrent_gated_delta_rule(*(d[n] for n in ("q", "k", "v", "g", "beta")), initial_state=d["S0"],
                                            output_final_state=True, **kw)


def cut(offsets, total):
    """What the offsets of a packed batch come down to: inside the tensors, never backwards."""
    out = []
    for c in offsets:
        out.append(max(out[-1] if out else 0, min(max(c, 0), total)))
    return out


# ------------------------------------------------------------------------ offsets that run backwards
@pytest.mark.parametrize("dtype,D", [(f32, 128), (f32, 64), (bf16, 32), (f32, 16), (bf16, 8)])
@pytest.mark.parametrize("offsets", [[0, 80, 60, 100], [0, 80, 60, 5000], [50, 0, 100], [-7, 20, -3, 20, 19, 90],
                                     [90, 10, 5, 0]])
def test_offsets_that_run_backwards_are_cut_in_a_forward_alone(offsets, dtype, D):
    T, N = 100, len(offsets) - 1
    d = make(1, T, 1, 2, D, dtype, seed=40, N=N)
    cu = torch.tensor(offsets, device=CUDA)
    f = lambda t: t.cpu().double()  # noqa: E731
    want_o, want_S = delta_rule_oracle(*(f(d[n]) for n in ("q", "k", "v", "g", "beta")), None, f(d["S0"]), cut(offsets, T))
    rtol = FP32_RTOL + (HALF_STEP if dtype == bf16 else 0)
    for o, S in (rule(d, cu=cu), recurrent(d, cu_seqlens=cu)):
        assert_close(o, want_o, rtol, "o", outlier_frac=0.0)
        assert_close(S, want_S, FP32_RTOL, "S")


def test_more_sequences_than_threads_order_their_offsets():
    """Every CTA takes the largest offset in front of its own sequence, however many there are."""
    gen = torch.Generator().manual_seed(41)
    offsets = torch.randint(0, 700, (600,), generator=gen).tolist()
    offsets[300:] = sorted(offsets[300:])
    T, N = 700, len(offsets) - 1
    d = make(1, T, 1, 1, 16, f32, seed=41, N=N)
    o, S = recurrent(d, cu_seqlens=torch.tensor(offsets, device=CUDA))
    leaves = {n: d[n].clone().requires_grad_(True) for n in ("v",)}
    o2, S2 = rule({**d, **leaves}, cu=torch.tensor(cut(offsets, T), device=CUDA))  # (the path that keeps ordered offsets)
    assert torch.equal(o, o2) and torch.equal(S, S2)


# ------------------------------------------------------------------------ launches beside another
def test_the_launch_in_front_of_one_that_runs_beside_it_is_ordinary():
    """In two parts: the pairs of the rest beside the first scan, the gradients of the rest beside the second reverse scan.  They
    read what earlier launches left without waiting, so the scan between must start when all of those have ended."""
    from test_launch_order_gpu import captured_launches
    d = make(2, 2200, 8, 16, 128, bf16, seed=42, state=False)
    leaves = {n: d[n].requires_grad_(True) for n in ("q", "k", "v", "g", "beta")}

    def step():
        o, _ = rule(d, final=False)
        return torch.autograd.grad(o, list(leaves.values()), d["do"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    kernels = [x for x in captured_launches(step) if "gdr_" in x.name]
    kinds = [next(k for k in ("pairs", "scan_bwd", "scan", "grad") if k in x.name) for x in kernels]
    assert kinds == ["pairs", "scan", "pairs", "scan", "scan_bwd", "scan_bwd", "grad", "grad"]
    assert not kernels[1].early and kernels[2].early and not kernels[5].early and kernels[6].early


# ------------------------------------------------------------------------ a wait that gives up
def test_the_status_word_is_this_calls():
    from delta_feedback_experiment_b200 import _lib, ops
    ops.track_device_status(True)  # (forgets the words of the calls before)
    assert _lib.native().last_status(False) is None and _lib.native().last_status(True) is None
    run_with_grads(make(2, 200, 2, 4, 128, bf16, seed=43))
    assert _lib.native().last_status(False) is not None and _lib.native().last_status(True) is not None
    assert ops.last_device_status() == 0 and ops.last_backward_status() == 0


@pytest.mark.parametrize("B,T,HK,HV,cu", [(2, 200, 2, 4, None), (2, 2200, 8, 16, None), (1, 300, 1, 3, [20, 21, 100, 280])],
                         ids=["whole", "two parts", "packed"])
def test_a_failure_reaches_every_result(B, T, HK, HV, cu):
    """Calls that start with the status word set, as a wait that gave up would leave it."""
    from delta_feedback_experiment_b200 import _lib, ops
    d = make(B, T, HK, HV, 128, bf16, seed=44, N=None if cu is None else len(cu) - 1)
    offsets = None if cu is None else torch.tensor(cu, device=CUDA)
    want = run_with_grads(d, offsets)
    ops.track_device_status(True)
    _lib.set_variant("gdr_scan", True)
    try:
        bad = run_with_grads(d, offsets)
        alone = rule(d, cu=offsets)
        assert ops.last_device_status() != 0 and ops.last_backward_status() != 0
    finally:
        _lib.set_variant("gdr_scan", False)
    starts = [0] if cu is None else cu[:-1]
    for o in (bad["o"], alone[0]):
        assert all(o[:, t].isnan().all() for t in starts)
    for S in (bad["S"], alone[1], bad["dS0"]):
        assert S.isnan().flatten(2).any(-1).all()
    for n in ("dq", "dk", "dv", "dg", "dbeta"):
        assert all(bad[n][:, t].isnan().any() for t in starts), n
    again = run_with_grads(d, offsets)
    assert [n for n in want if not torch.equal(want[n], again[n])] == []
    assert ops.last_device_status() == 0 and ops.last_backward_status() == 0


# ------------------------------------------------------------------------ derivatives
def test_a_missing_second_derivative_is_not_silent():
    d = make(1, 20, 1, 1, 64, f32, seed=45)
    g = d["g"].clone().requires_grad_(True)
    o, _ = rule({**d, "g": g})
    with pytest.warns(UserWarning, match="differentiable once"):
        (dg,) = torch.autograd.grad(o.sum(), g, create_graph=True)
    with pytest.raises(RuntimeError, match="does not require grad"):
        dg.sum().backward()


def test_a_first_derivative_does_not_warn(recwarn):
    run_with_grads(make(1, 20, 1, 1, 64, f32, seed=45))
    assert not [w for w in recwarn if "differentiable" in str(w.message)]


def test_forward_mode_raises():
    from torch.autograd import forward_ad
    d = make(1, 20, 1, 1, 64, f32, seed=46)
    with forward_ad.dual_level():
        v = forward_ad.make_dual(d["v"], torch.ones_like(d["v"]))
        with pytest.raises(RuntimeError, match="jvp"):
            rule({**d, "v": v})
