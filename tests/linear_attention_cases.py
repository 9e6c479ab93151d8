"""Seeded inputs and tolerances of the linear-attention tests."""

import torch

from conftest import assert_close
from oracle.linear_attention_oracle import attend_with_grads

# fp32 arithmetic: a number passes up to T roundings of 2^-24 on its way through the state, in both directions of a
# gradient, and sums of some hundred terms add theirs: 2 * 512 * 2^-24 = 6e-5.
FP32_RTOL = 1e-4
# Chunked kernels (bf16 activations of 128 and 64 channels): computed operands are two bf16 parts, off by at most 2^-16
# (2^-17 of the number and the rounding of what is left), two of them in a row for what passes through a state.  fp32
# results: that, relative to an entry or to the root mean square around it.
SPLIT = 2.0 ** -15
# bf16 results: their own rounding, half a step, and the above.
HALF_STEP = 2.0 ** -8
# The gate's gradient of the chunked kernels is a difference of sums (``gate_bound``).
NAMES = ("q", "k", "v", "g")


def make(B, T, HK, HV, D, dtype, seed, N=None, state=True, gate="token", strength=0.3, device="cuda"):
    """Inputs on the CPU's generator (the same everywhere), ``[B,T,...]``; N states."""
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)  # noqa: E731
    N = B if N is None else N
    g = -torch.nn.functional.softplus(n(B, T, HV) if gate == "token" else n(HV)) * strength
    if gate == "strong":
        g = -torch.nn.functional.softplus(n(B, T, HV)) * torch.linspace(0.02, 12, HV)
    d = {"q": unit(n(B, T, HK, D)).to(dtype), "k": unit(torch.nn.functional.silu(n(B, T, HK, D))).to(dtype),
         "v": n(B, T, HV, D).to(dtype), "g": g, "do": n(B, T, HV, D).to(dtype),
         "dS": n(N, HV, D, D) * 0.3 if state else None, "S0": n(N, HV, D, D) * 0.3 if state else None}
    return {k: None if t is None else t.to(device) for k, t in d.items()}


def attend(d, cu=None, final=True, **kw):
    from delta_feedback_experiment_b200 import chunk_linear_attention
    return chunk_linear_attention(*(d[n] for n in NAMES), initial_state=d["S0"], output_final_state=final,
                                  cu_seqlens=cu, **kw)


def run_with_grads(d, cu=None, scale=None):
    leaves = {n: d[n].detach().clone().requires_grad_(True) for n in (*NAMES, "S0") if d[n] is not None}
    o, S = attend({**d, **leaves}, cu=cu, scale=scale)
    outs, cots = ([o, S], [d["do"], d["dS"]]) if d["dS"] is not None else ([o], [d["do"]])
    grads = torch.autograd.grad(outs, list(leaves.values()), cots)
    return {"o": o.detach(), "S": S.detach(), **{"d" + n: t for n, t in zip(leaves, grads)}}


def expected(d, cu=None, scale=None):
    return attend_with_grads(d, cu, scale)


def gate_bound(d, want, cu=None):
    """How far the chunked kernels' gradient of the gate may be off, beside the rounding of the result.

    ``dg_t = sum_{u >= t} (row_u - col_u) + <S_end, dS_end>`` with ``row_u = q_u.dq_u = do_u.o_u`` and ``col_u = k_u.dk_u =
    v_u.dv_u`` of the head.  A row or a column is a product of one computed operand, off by at most 2^-16 (two bf16 parts of it, and of
    the state it was made from), so it is off by at most that; the errors of different tokens have nothing to do with one another and
    add up like a random walk, root mean square at most ``2^-16 sqrt(sum (row^2 + col^2))`` over the sequence.  Twice that is asked
    for (a single one is 2^-19 in the mean).  The gradient of one decay a head adds ``dg_t`` over t: token u's error counts once for
    each token up to it."""
    row, col = (d["do"].double().cpu() * want["o"]).sum(-1), (d["v"].double().cpu() * want["dv"]).sum(-1)
    power = row.square() + col.square()                                      # [B, T, HV]
    B, T = power.shape[:2]
    spans = [(b, 0, T) for b in range(B)] if cu is None else [(0, int(s), int(e)) for s, e in zip(cu, cu[1:])]
    each, whole = torch.zeros_like(power), torch.zeros(power.shape[2], dtype=torch.float64)
    for b, s, e in spans:
        each[b, s:e] = power[b, s:e].sum(0).sqrt()
        count = torch.arange(1, e - s + 1, dtype=torch.float64)[:, None]
        whole += (count.square() * power[b, s:e]).sum(0)
    return 2.0 ** -15 * (whole.sqrt() if d["g"].dim() == 1 else each)


def check(got, want, d, cu=None, where=""):
    assert set(got) == set(want), (set(got), set(want))
    chunked = got["o"].dtype == torch.bfloat16 and got["o"].shape[-1] >= 64
    for name, t in got.items():
        if chunked and name == "dg":
            e = want[name]
            bound = gate_bound(d, want, cu) + SPLIT * (e.abs() + e.square().mean().sqrt())
            worst = ((t.double().cpu() - e).abs() / bound).nan_to_num(0.0, posinf=9e9).max() if t.numel() else 0.0
            assert t.isfinite().all() and worst <= 1.0, f"{where}:dg off by {float(worst):.3f} of what it may be"
            continue
        rtol = SPLIT if chunked else FP32_RTOL
        if t.dtype == torch.bfloat16:
            rtol += HALF_STEP
        assert_close(t, want[name], rtol, f"{where}:{name}", outlier_frac=0.0)
