"""Seeded inputs and tolerances of the gated delta rule's tests."""

import torch

from conftest import assert_close
from oracle.delta_rule_oracle import delta_rule_with_grads

FP32_RTOL = 1e-4      # fp32 arithmetic of a few hundred dependent tokens against 64 bits
BF16_RTOL = 2e-2      # chunked kernels: state, keys' correction, writes, T and pair matrices are rounded to bf16 on the way to
#                       an output and its own rounding: 6 x 2^-8 = 2.3e-2 if all were at their worst and lined up
HALF_STEP = 2.0 ** -8  # rounding of an output to bf16


def make(B, T, HK, HV, D, dtype, seed, N=None, state=True, strong=False, device="cuda"):
    """Inputs on the CPU's generator (the same everywhere), ``[B,T,...]``; N states."""
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)  # noqa: E731
    N = B if N is None else N
    g = -torch.nn.functional.softplus(n(B, T, HV)) * (torch.linspace(0.02, 12, HV) if strong else 0.3)
    d = {"q": unit(n(B, T, HK, D)).to(dtype), "k": unit(torch.nn.functional.silu(n(B, T, HK, D))).to(dtype),
         "v": n(B, T, HV, D).to(dtype), "g": g, "beta": torch.sigmoid(n(B, T, HV)).to(dtype),
         "do": n(B, T, HV, D).to(dtype), "dS": n(N, HV, D, D) * 0.3 if state else None,
         "S0": n(N, HV, D, D) * 0.3 if state else None}
    return {k: None if t is None else t.to(device) for k, t in d.items()}


def rule(d, names=("q", "k", "v", "g", "beta"), cu=None, final=True, **kw):
    from delta_feedback_experiment_b200 import chunk_gated_delta_rule
    return chunk_gated_delta_rule(*(d[n] for n in names), initial_state=d["S0"], output_final_state=final,
                                  cu_seqlens=cu, **kw)


def run_with_grads(d, cu=None, scale=None):
    leaves = {n: d[n].detach().clone().requires_grad_(True) for n in ("q", "k", "v", "g", "beta", "S0")
              if d[n] is not None}
    o, S = rule({**d, **leaves}, cu=cu, scale=scale)
    outs, cots = ([o, S], [d["do"], d["dS"]]) if d["dS"] is not None else ([o], [d["do"]])
    grads = torch.autograd.grad(outs, list(leaves.values()), cots)
    return {"o": o.detach(), "S": S.detach(), **{"d" + n: t for n, t in zip(leaves, grads)}}


def expected(d, cu=None, scale=None):
    return delta_rule_with_grads([d[n] for n in ("q", "k", "v", "g", "beta")], d["do"], d["dS"], scale,
                                 d["S0"], cu)


def check(got, want, chunked, where=""):
    assert set(got) == set(want), (set(got), set(want))
    for name, t in got.items():
        rtol = BF16_RTOL if chunked else FP32_RTOL
        if not chunked and t.dtype == torch.bfloat16:
            rtol += HALF_STEP
        assert_close(t, want[name], rtol, f"{where}:{name}", outlier_frac=1e-4 if chunked else 0.0)
