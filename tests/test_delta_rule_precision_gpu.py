"""How near the chunked kernels (bf16 heads of 128 channels) come to the definition in 64 bits.

Every operand that they compute is split in two bf16 parts, off by at most u = 2^-18 of the value, and a product of two
such operands leaves the product of the lo parts out, u again.  A state takes six of these errors a chunk (state, correction
and T as operands, T's own split, the write, the product that is left out), and chunks hand them on decayed: at most 8 u of
the states' root mean square.  A gate's gradient sums products of two results of that kind (16 u) and of a pair matrix
that is split again: 24 u.  A result that leaves as bf16 is off by half a step, 2^-8 of it, and by what it had before: 8 u root
mean square at most, 48 u for any one of 2^18 entries (five to six deviations).  With one lo part missing anywhere the
errors would be near 2^-10 = 256 u."""

import pytest
import torch

from conftest import assert_close, rel_rms
from delta_rule_cases import FP32_RTOL, HALF_STEP, expected, make, run_with_grads

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16
U = 2.0 ** -18
RMS_BOUND = {"S": 8 * U, "dS0": 8 * U, "dg": 24 * U}
ENTRY_BOUND = 48 * U


def beyond_its_rounding(actual, want):
    """The largest part of an entry's error that its rounding does not explain, in units of |entry| + root mean square
    (of its row or of all, the larger)."""
    a, e = actual.double().cpu(), want.double()
    rms = e.square().mean().sqrt()
    if e.ndim == 4:
        rms = torch.maximum(rms, e.square().mean(-1, keepdim=True).sqrt())
    return float((((a - e).abs() - HALF_STEP * e.abs()) / (e.abs() + rms)).max())


@pytest.mark.parametrize("strong", [False, True], ids=["mild", "strong"])
@pytest.mark.parametrize("B,T,HK,HV,cu", [
    (1, 64, 1, 1, None), (2, 65, 1, 3, None), (1, 517, 1, 2, None), (1, 1100, 2, 2, None), (1, 300, 2, 4, [0, 1, 70, 70, 290])])
def test_outputs_are_off_by_their_rounding_alone(B, T, HK, HV, cu, strong):
    d = make(B, T, HK, HV, 128, bf16, seed=7 * T + HV, N=None if cu is None else len(cu) - 1, strong=strong)
    got = run_with_grads(d, None if cu is None else torch.tensor(cu, device="cuda"))
    want = expected(d, cu)
    off = {n: rel_rms(got[n], want[n]) / U for n in RMS_BOUND}
    off.update({n: beyond_its_rounding(got[n], want[n]) / U for n in ("o", "dq", "dk", "dv", "dbeta")})
    bounds = {n: RMS_BOUND.get(n, ENTRY_BOUND) / U for n in off}
    assert all(off[n] <= bounds[n] for n in off), {n: (round(off[n], 2), bounds[n]) for n in off if off[n] > bounds[n]}


# ------------------------------------------------------------------------ write strengths in fp32 beside bf16 activations
@pytest.mark.parametrize("cu", [None, [4, 70, 70, 230]], ids=["dense", "packed"])
def test_write_strengths_in_fp32_are_not_rounded(cu):
    """Rounded to bf16 they would move states by 2^-9 of every write.  Their gradient is a product of two chunked results
    (16 u, and u for the product that is left out) and stays in fp32."""
    d = make(1, 240, 2, 4, 128, bf16, seed=5, N=None if cu is None else len(cu) - 1)
    d["beta"] = (d["beta"].float() * 0.999 + 0.0005)
    if cu is not None:
        d["beta"][:, :cu[0]] = float("nan")
    got = run_with_grads(d, None if cu is None else torch.tensor(cu, device="cuda"))
    want = expected({**d, "beta": d["beta"].nan_to_num()}, cu)
    assert got["dbeta"].dtype == torch.float32
    off = {n: rel_rms(got[n], want[n]) / U for n in RMS_BOUND} | {"dbeta": rel_rms(got["dbeta"], want["dbeta"]) / U}
    assert all(off[n] <= (RMS_BOUND.get(n, 24 * U)) / U for n in off), off
    if cu is not None:
        assert (got["dbeta"][:, :cu[0]] == 0).all() and (got["dbeta"][:, cu[-1]:] == 0).all()


@pytest.mark.parametrize("T,D", [(1, 128), (2, 16), (5, 128), (70, 64), (33, 8)])
def test_write_strengths_in_fp32_in_the_exact_kernels(T, D):
    from delta_feedback_experiment_b200 import fused_recurrent_gated_delta_rule
    d = make(2, T, 1, 2, D, bf16, seed=6)
    d["beta"] = (d["beta"].float() * 0.999 + 0.0005)
    want = expected(d)
    _, S = fused_recurrent_gated_delta_rule(*(d[n] for n in ("q", "k", "v", "g", "beta")), initial_state=d["S0"],
                                            output_final_state=True)
    assert_close(S, want["S"], FP32_RTOL, "S")
    if D < 128:
        got = run_with_grads(d)
        assert got["dbeta"].dtype == torch.float32
        for n in ("S", "dbeta", "dg", "dS0"):
            assert_close(got[n], want[n], FP32_RTOL, n)
