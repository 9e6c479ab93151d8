"""Linear attention with a decay for each head and the norm and rotation of queries and keys, from their
definitions in 64 bits (gradients by autograd)."""

import torch


def attend(q, k, v, g, scale=None, S0=None, cu=None):
    """``q``, ``k`` ``[B,T,HK,D]``, ``v`` ``[B,T,HV,D]``, ``g`` ``[B,T,HV]`` or ``[HV]`` -> ``o``, ``S`` ``[N,HV,D,D]``,
    token by token.  ``cu`` (a list of offsets): sequences of one row; rows that none owns give zeros."""
    B, T, HV, D = v.shape
    scale = D ** -0.5 if scale is None else scale
    q, k = (t.repeat_interleave(HV // t.shape[2], 2) for t in (q, k))
    a = g.exp().expand(B, T, HV)
    spans = [(b, 0, T) for b in range(B)] if cu is None else [(0, s, e) for s, e in zip(cu, cu[1:])]
    rows = {}
    states = []
    for n, (b, s, e) in enumerate(spans):
        S = v.new_zeros(HV, D, D) if S0 is None else S0[n]
        for t in range(s, e):
            S = a[b, t, :, None, None] * S + k[b, t, :, :, None] * v[b, t, :, None, :]
            rows[b, t] = scale * (S * q[b, t, :, :, None]).sum(1)
        states.append(S)
    zero = v.new_zeros(HV, D)
    o = torch.stack([torch.stack([rows.get((b, t), zero) for t in range(T)]) for b in range(B)]) if T else v * 1.0
    return o, torch.stack(states) if states else v.new_zeros(0, HV, D, D)


def attend_with_grads(d, cu=None, scale=None):
    """Values and gradients for the inputs of a dict: q, k, v, g, S0 (or None), do, dS (or None)."""
    x = {n: d[n].detach().double().cpu().requires_grad_(True) for n in ("q", "k", "v", "g", "S0") if d[n] is not None}
    o, S = attend(x["q"], x["k"], x["v"], x["g"], scale, x.get("S0"), None if cu is None else [int(c) for c in cu])
    loss = (o * d["do"].double().cpu()).sum()
    if d["dS"] is not None:
        loss = loss + (S * d["dS"].double().cpu()).sum()
    grads = torch.autograd.grad(loss, list(x.values()), allow_unused=True)
    out = {"o": o.detach(), "S": S.detach()}
    for (n, t), dt in zip(x.items(), grads):
        out["d" + n] = torch.zeros_like(t) if dt is None else dt
    return out


def norm_rotate(x, weight=None, inv_freq=None, positions=None, eps=1e-6, interleaved=False):
    """``x`` ``[B,T,H,D]`` in fp64; ``positions`` ``[B,T]`` or ``[T]``."""
    B, T, _, D = x.shape
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        y = y * weight
    if inv_freq is None or not inv_freq.numel():
        return y
    at = torch.arange(T) if positions is None else positions
    angle = at.double().expand(B, T)[..., None, None] * inv_freq.double()
    half = inv_freq.numel()
    a, b = (y[..., :2 * half:2], y[..., 1:2 * half:2]) if interleaved else (y[..., :half], y[..., half:2 * half])
    a, b = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1)
