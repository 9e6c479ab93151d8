"""Linear attention in 64 bits, chunk by chunk with autograd, for rows too long for the oracle's token by token (which it is held
to in ``test_linear_attention_chunks64.py``)."""

import torch

CHUNK = 64


def attend(q, k, v, g, scale, S0, spans):
    """``[B,T,H,D]`` rows in fp64 (keys and queries of each value head), ``g`` ``[B,T,H]``; spans of ``(row, start, end)`` -> ``o``, ``S``."""
    H, D = v.shape[2:]
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=v.device).tril()
    rows, states = {b: [] for b in range(v.shape[0])}, []
    at = dict.fromkeys(rows, 0)

    def gap(b, end):  # rows that no span owns
        if end > at[b]:
            rows[b].append(v.new_zeros(H, end - at[b], D))

    for n, (b, start, end) in enumerate(spans):
        gap(b, start)
        S = v.new_zeros(H, D, D) if S0 is None else S0[n]
        for t in range(start, end, CHUNK):
            x, y, z, e = (w[b, t:min(t + CHUNK, end)].movedim(1, 0) for w in (q, k, v, g))
            G = e.cumsum(-1)
            m = low[:G.shape[1], :G.shape[1]]
            pairs = (x @ y.transpose(1, 2)) * (G[:, :, None] - G[:, None, :]).masked_fill(~m, -torch.inf).exp()
            rows[b].append(scale * (pairs @ z + (x * G.exp()[..., None]) @ S))
            S = S * G[:, -1].exp()[:, None, None] + (y * (G[:, -1:] - G).exp()[..., None]).transpose(1, 2) @ z
        states.append(S)
        at[b] = max(end, at[b])
    for b in rows:
        gap(b, v.shape[1])
    o = torch.stack([torch.cat(rows[b], 1).movedim(0, 1) for b in rows])
    return o, torch.stack(states)


def attend_with_grads(d, cu=None, scale=None):
    """As the oracle's, on the device of the inputs."""
    x = {n: d[n].detach().double().requires_grad_(True) for n in ("q", "k", "v", "g", "S0") if d[n] is not None}
    B, T, HV, D = d["v"].shape
    q, k = (x[n].repeat_interleave(HV // d[n].shape[2], 2) for n in ("q", "k"))
    spans = [(b, 0, T) for b in range(B)] if cu is None else [(0, int(s), int(e)) for s, e in zip(cu, cu[1:])]
    o, S = attend(q, k, x["v"], x["g"].expand(B, T, HV), D ** -0.5 if scale is None else scale, x.get("S0"), spans)
    loss = (o * d["do"].double()).sum()
    if d["dS"] is not None:
        loss = loss + (S * d["dS"].double()).sum()
    grads = torch.autograd.grad(loss, list(x.values()))
    return {"o": o.detach().cpu(), "S": S.detach().cpu(), **{"d" + n: t.cpu() for n, t in zip(x, grads)}}
