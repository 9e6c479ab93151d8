"""CPU definitions of the gated delta rule and of layer norm, token by token and row by row, in
the dtype of the given tensors (fp64 in the tests); autograd supplies the gradients."""

from __future__ import annotations

import torch


def delta_rule_oracle(q, k, v, g, beta, scale=None, initial_state=None, cu_seqlens=None):
    """``[B,T,HK,D]`` q and k, ``[B,T,HV,D]`` v -> ``(o, final_state)``.  Packed rows (a list of
    offsets) one sequence after the other; rows outside every sequence give zeros."""
    B, T, HK, D = q.shape
    HV = v.shape[2]
    scale = D ** -0.5 if scale is None else scale
    if cu_seqlens is not None:
        o, states, ends = [], [], [int(c) for c in cu_seqlens]
        zero = lambda n: v.new_zeros(1, n, HV, D)  # noqa: E731
        o.append(zero(ends[0]))
        for i, (a, b) in enumerate(zip(ends[:-1], ends[1:])):
            S0 = None if initial_state is None else initial_state[i:i + 1]
            part = [t[:, a:b] for t in (q, k, v, g, beta)]
            oi, Si = delta_rule_oracle(*part, scale, S0)
            o.append(oi)
            states.append(Si)
        o.append(zero(T - ends[-1]))
        return torch.cat(o, 1), torch.cat(states) if states else v.new_zeros(0, HV, D, D)
    q, k = (t.repeat_interleave(HV // HK, 2) for t in (q, k))
    S = v.new_zeros(B, HV, D, D) if initial_state is None else initial_state
    out = []
    for t in range(T):
        S = S * g[:, t].exp()[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - torch.einsum("bhk,bhkv->bhv", k[:, t], S))
        S = S + k[:, t, :, :, None] * u[:, :, None, :]
        out.append(scale * torch.einsum("bhk,bhkv->bhv", q[:, t], S))
    return torch.stack(out, 1) if out else torch.zeros_like(v), S


def delta_rule_with_grads(inputs, do, dS=None, scale=None, initial_state=None, cu_seqlens=None,
                          dtype=torch.float64):
    """Outputs and gradients as a dict: o, S, dq, dk, dv, dg, dbeta (dS0 with an initial state)."""
    x = [t.detach().cpu().to(dtype).requires_grad_(True) for t in inputs]
    S0 = None if initial_state is None else initial_state.detach().cpu().to(dtype).requires_grad_(True)
    o, S = delta_rule_oracle(*x, scale, S0, cu_seqlens)
    loss = (o * do.cpu().to(dtype)).sum()
    if dS is not None:
        loss = loss + (S * dS.cpu().to(dtype)).sum()
    leaves = x + ([S0] if S0 is not None else [])
    grads = torch.autograd.grad(loss, leaves, allow_unused=True)
    grads = [torch.zeros_like(leaf) if d is None else d for leaf, d in zip(leaves, grads)]
    names = ["dq", "dk", "dv", "dg", "dbeta", "dS0"]
    return {"o": o.detach(), "S": S.detach(), **dict(zip(names, grads))}


def layer_norm_oracle(x, weight=None, bias=None, eps=1e-5):
    c = x - x.mean(-1, keepdim=True)
    y = c / (c.square().mean(-1, keepdim=True) + eps).sqrt()
    y = y if weight is None else y * weight
    return y if bias is None else y + bias
