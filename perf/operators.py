"""The gated delta rule (chunked and recurrent) and layer norm: what is timed, and what it must return.

A case is one call a host makes: a cached decoding step, the prefill of a prompt, the forward +
backward of a training step (dense or packed), or a layer norm.  ``listed()`` names representative
cases, ``draw()`` gives more of the same ranges.

The gated delta rule, per value head with state ``S [K, V]`` and key head ``h // (HV / HK)``:

    S_t = a_t S_{t-1} + k_t u_t^T,   a_t = exp(g_t),   u_t = beta_t (v_t - a_t S_{t-1}^T k_t),
    o_t = scale S_t^T q_t.

``run`` computes it in plain torch, 64 tokens at a time in 32 bits, or calls the framework's
operators; ``exact`` goes token by token in 64 bits with the reverse recurrence written out.
"""

from __future__ import annotations

import math
import random

import torch

own = False

CHUNK = 64
LN_EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # One user, one token: the latency of a cached decoding step of a small layer.
        {"name": "rule-decode-1", "kind": "recurrent", "B": 1, "T": 1, "HK": 8, "HV": 8, "D": 128, "dtype": "bf16",
         "dist": "production"},
        # 256 users, 32 heads with shared keys: 512 MB of state read and written.
        {"name": "rule-decode-256", "kind": "recurrent", "B": 256, "T": 1, "HK": 16, "HV": 32, "D": 128,
         "dtype": "bf16", "dist": "production"},
        # A few tokens appended to cached rows (a short prompt, a speculative block).
        {"name": "rule-append-48", "kind": "recurrent", "B": 4, "T": 48, "HK": 16, "HV": 16, "D": 128, "dtype": "bf16",
         "dist": "production"},
        # One long prompt of odd length: forward only, the final state is kept.
        {"name": "rule-prefill-8191", "kind": "prefill", "B": 1, "T": 8191, "HK": 16, "HV": 16, "D": 128,
         "dtype": "bf16", "dist": "production", "state": False},
        # The headline training shape.
        {"name": "rule-train", "kind": "train", "B": 8, "T": 4096, "HK": 16, "HV": 16, "D": 128, "dtype": "bf16",
         "dist": "unit", "state": False},
        # Value heads that share key heads, states in and out, a ragged length.
        {"name": "rule-train-shared", "kind": "train", "B": 2, "T": 2047, "HK": 4, "HV": 12, "D": 128, "dtype": "bf16",
         "dist": "production", "state": True},
        # Documents of 17 to 4,096 tokens packed to one row.
        {"name": "rule-packed", "kind": "packed", "total": 32768, "lo": 17, "hi": 4096, "cut": 7, "HK": 8, "HV": 16,
         "D": 128, "dtype": "bf16", "dist": "production", "state": True},
        # The fp32 configuration, heads of 64 channels.
        {"name": "rule-exact", "kind": "train", "B": 2, "T": 512, "HK": 4, "HV": 4, "D": 64, "dtype": "fp32",
         "dist": "unit", "state": True},
        # Layer norm of a training step: 32,768 rows of 2,048 channels, weight and bias.
        {"name": "norm-train", "kind": "norm", "rows": 32768, "dim": 2048, "dtype": "bf16", "affine": True,
         "grad": True},
        # Rows of an odd width that no vector load divides, in fp32.
        {"name": "norm-odd", "kind": "norm", "rows": 1001, "dim": 1003, "dtype": "fp32", "affine": True, "grad": True},
        # Wide rows.
        {"name": "norm-wide", "kind": "norm", "rows": 1024, "dim": 16384, "dtype": "bf16", "affine": True,
         "grad": True},
        # The norm of a decoding step: a few rows, forward only.
        {"name": "norm-decode", "kind": "norm", "rows": 8, "dim": 2048, "dtype": "bf16", "affine": True,
         "grad": False},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_UNITS = 8 * 4096 * 16       # (token, value head) pairs of a drawn case, at most
HEADS = ((1, 1), (2, 2), (4, 4), (8, 8), (16, 16), (2, 8), (4, 12), (8, 16), (16, 32))


def draw(rng: random.Random):
    kind = rng.choice(("recurrent", "recurrent", "prefill", "train", "train", "train", "packed", "norm", "norm"))
    if kind == "norm":
        dim = _log(rng, 8, 16384)
        if rng.random() < 0.6:
            dim = max(8, dim // 8 * 8)
        return {"kind": kind, "rows": _log(rng, 1, min(32768, 32768 * 2048 // dim)), "dim": dim,
                "dtype": rng.choice(("bf16", "bf16", "fp32")), "affine": rng.random() < 0.8,
                "grad": rng.random() < 0.7}
    HK, HV = rng.choice(HEADS)
    dtype, D = rng.choice((("bf16", 128), ("bf16", 128), ("bf16", 128), ("bf16", 64), ("fp32", 64), ("fp32", 128),
                           ("fp32", 32)))
    c = {"kind": kind, "HK": HK, "HV": HV, "D": D, "dtype": dtype, "dist": rng.choice(("unit", "production"))}
    if kind == "recurrent":
        T = rng.choice((1, 1, 1, 2, 5, 16, 33, 64))
        c.update(B=_log(rng, 1, max(1, 8192 // (HV * T))), T=T)
        return c
    fast = dtype == "bf16" and D == 128
    c["state"] = rng.random() < 0.5
    if kind == "packed":
        hi = rng.choice((200, 1024, 4096))
        most = 2048 if not fast else 8192 if hi == 200 else min(32768, MOST_UNITS // HV)
        c.update(total=_log(rng, 256, most), lo=rng.choice((1, 17, 128)), hi=hi, cut=rng.randrange(1000))
        return c
    T = _log(rng, 1, 8192 if fast else 1024)
    c.update(T=T, B=_log(rng, 1, max(1, min(16, (MOST_UNITS if fast else 16384) // (T * HV)))))
    return c


def _lengths(case):
    """Sequence lengths of a packed case: uniform in [lo, hi], the last one cut to the total."""
    rng, left, out = random.Random(case["cut"]), case["total"], []
    while left:
        out.append(min(left, rng.randint(case["lo"], case["hi"])))
        left -= out[-1]
    return out


# ------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def n(*size):
        return torch.randn(size, generator=gen, device="cuda")

    def u(lo, hi, *size):
        return torch.rand(size, generator=gen, device="cuda") * (hi - lo) + lo

    dt = DTYPES[case["dtype"]]
    if case["kind"] == "norm":
        R, N = case["rows"], case["dim"]
        s = {"kind": "norm", "x": (n(R, N) * 1.5 + 0.3).to(dt), "grad": case["grad"], "weight": None, "bias": None}
        if case["affine"]:
            s["weight"], s["bias"] = 1 + 0.2 * n(N), 0.2 * n(N)
        if case["grad"]:
            s["dy"] = n(R, N).to(dt)
        return s
    packed = case["kind"] == "packed"
    lens = _lengths(case) if packed else None
    B, T = (1, case["total"]) if packed else (case["B"], case["T"])
    HK, HV, D = case["HK"], case["HV"], case["D"]
    N = len(lens) if packed else B
    silu = torch.nn.functional.silu
    unit = case["dist"] == "unit"
    norm = lambda t: t / t.square().sum(-1, keepdim=True).add(1e-6).sqrt()  # noqa: E731
    # keys and queries as a short convolution with SiLU and a norm leaves them, or evenly spread ones
    q, k = (norm(n(B, T, HK, D) if unit else silu(n(B, T, HK, D))).to(dt) for _ in range(2))
    v = (n(B, T, HV, D) if unit else silu(n(B, T, HV, D))).to(dt)
    if unit:
        g = -torch.nn.functional.softplus(n(B, T, HV))
    else:  # exp(A_log) ~ U(1, 16) and steps of 1e-3 to 1e-1, as such layers are initialised
        step = u(math.log(1e-3), math.log(1e-1), HV).exp()
        bias = step + torch.log(-torch.expm1(-step))
        g = -u(1.0, 16.0, HV) * torch.nn.functional.softplus(0.5 * n(B, T, HV) + bias)
    s = {"kind": case["kind"], "q": q, "k": k, "v": v, "g": g, "beta": torch.sigmoid(n(B, T, HV)).to(dt),
         "scale": D ** -0.5, "S0": None, "lens": lens, "cu": None}
    if case["kind"] == "recurrent" or case["state"]:
        s["S0"] = 0.1 * n(N, HV, D, D)
    if packed:
        ends = [0]
        for length in lens:
            ends.append(ends[-1] + length)
        s["cu"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    if case["kind"] in ("train", "packed"):
        s["do"] = n(B, T, HV, D).to(dt)
        if case["state"]:
            s["dS"] = 0.1 * n(N, HV, D, D)
    return s


# -------------------------------------------------------------------- plain forms
def _plain_step(q, k, v, g, beta, scale, S):
    """One token: [B, HV, D] rows on S [B, HV, D, D], everything fp32."""
    S = S * g.exp()[..., None, None]
    u = beta[..., None] * (v - (S * k[..., None]).sum(-2))
    S = S + k[..., None] * u[..., None, :]
    return scale * (S * q[..., None]).sum(-2), S


def _plain_rule(q, k, v, g, beta, scale, S):
    """``[N, T, H, D]`` fp32 rows (keys and queries repeated to the value heads), state or None ->
    output and final state, a chunk of 64 tokens at a time."""
    N, T, H, D = v.shape
    NC = -(-T // CHUNK)
    pad = NC * CHUNK - T

    def cut(t):  # [N, T, H, ...] -> [N, H, NC, 64, ...]; added rows are zero and leave the state alone
        if pad:
            t = torch.cat((t, t.new_zeros(N, pad, *t.shape[2:])), 1)
        return t.reshape(N, NC, CHUNK, *t.shape[2:]).movedim(3, 1)

    q, k, v, g, b = (cut(t) for t in (q, k, v, g, beta))
    G = g.cumsum(-1)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=v.device).tril()
    decay = (G[..., :, None] - G[..., None, :]).masked_fill(~low, -math.inf).exp()
    P = scale * (q @ k.transpose(-1, -2)) * decay
    L = ((k @ k.transpose(-1, -2)) * decay).masked_fill(~low.tril(-1), 0.0) * b[..., None, :]
    eye = torch.eye(CHUNK, device=v.device)
    with torch.no_grad():  # (I + L)^-1 row by row
        T0 = eye.expand_as(L).contiguous()
        for i in range(1, CHUNK):
            T0[..., i, :i] = -(L[..., i:i + 1, :i] @ T0[..., :i, :i])[..., 0, :]
    # one refinement step, which also carries the derivative: d(T0 (I - (I + L) T0)) = -T0 dL T0
    Ti = T0 + T0 @ (eye - (eye + L) @ T0)
    W, U = Ti @ (G.exp()[..., None] * k), Ti @ v
    kd = k * (G[..., -1:] - G).exp()[..., None]
    qd = scale * q * G.exp()[..., None]
    S = v.new_zeros(N, H, D, D) if S is None else S
    o = []
    for c in range(NC):
        u = b[:, :, c, :, None] * (U[:, :, c] - W[:, :, c] @ S)
        o.append(qd[:, :, c] @ S + P[:, :, c] @ u)
        S = S * G[:, :, c, -1, None, None].exp() + kd[:, :, c].transpose(-1, -2) @ u
    return torch.stack(o, 2).movedim(1, 3).reshape(N, NC * CHUNK, H, D)[:, :T], S


def _plain(s):
    dt, HK, HV = s["v"].dtype, s["k"].shape[2], s["v"].shape[2]
    grad = "do" in s
    names = ["q", "k", "v", "g", "beta"] + (["S0"] if s["S0"] is not None else [])
    x = {n: s[n].float().requires_grad_(grad) for n in names}
    wide = {n: x[n].repeat_interleave(HV // HK, 2) for n in ("q", "k")}
    rows = [wide["q"], wide["k"], x["v"], x["g"], x["beta"]]
    S0 = x.get("S0")
    with torch.set_grad_enabled(grad):
        if s["lens"] is not None:  # sequences as rows of one batch, zero rows behind the short ones
            lens = s["lens"]
            most = max(lens)
            at = torch.arange(most, device="cuda")
            n = torch.tensor(lens, device="cuda")
            start = n.cumsum(0) - n
            real = at < n[:, None]
            index = torch.where(real, start[:, None] + at, 0)
            rows = [t[0][index] * real.reshape(*real.shape, *[1] * (t.ndim - 2)) for t in rows]
            o, S = _plain_rule(*rows, s["scale"], S0)
            o = o[real][None]
        elif s["v"].shape[1] == 1:
            o, S = _plain_step(*(t[:, 0] for t in rows), s["scale"], S0 if S0 is not None else 0.0)
            o = o[:, None]
        else:
            o, S = _plain_rule(*rows, s["scale"], S0)
    if not grad:
        return [o.to(dt), S]
    outs, cots = ([o, S], [s["do"].float(), s["dS"]]) if "dS" in s else ([o], [s["do"].float()])
    grads = torch.autograd.grad(outs, list(x.values()), cots)
    return [o.detach().to(dt), S.detach()] + [d.to(s[n].dtype) for n, d in zip(names, grads)]


def _plain_norm(s):
    grad, dt = s["grad"], s["x"].dtype
    x = s["x"].float().requires_grad_(grad)
    affine = s["weight"] is not None
    w, b = (s[n].detach().clone().requires_grad_(grad) if affine else None for n in ("weight", "bias"))
    with torch.set_grad_enabled(grad):
        c = x - x.mean(-1, keepdim=True)
        y = c * (c.square().mean(-1, keepdim=True) + LN_EPS).rsqrt()
        if affine:
            y = y * w + b
    if not grad:
        return [y.to(dt)]
    leaves = [x, w, b] if affine else [x]
    d = torch.autograd.grad(y, leaves, s["dy"].float())
    return [y.detach().to(dt), d[0].to(dt), *d[1:]]


# ------------------------------------------------------------- the framework's calls
def _own(s):
    from delta_feedback_experiment_b200 import chunk_gated_delta_rule, fused_recurrent_gated_delta_rule
    if s["kind"] == "recurrent":
        o, S = fused_recurrent_gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], scale=s["scale"],
                                                initial_state=s["S0"], output_final_state=True)
        return [o, S]
    grad = "do" in s
    names = ["q", "k", "v", "g", "beta"] + (["S0"] if s["S0"] is not None else [])
    x = {n: s[n].detach().requires_grad_(grad) for n in names}
    o, S = chunk_gated_delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], scale=s["scale"],
                                  initial_state=x.get("S0"), output_final_state=True, cu_seqlens=s["cu"])
    if not grad:
        return [o, S]
    outs, cots = ([o, S], [s["do"], s["dS"]]) if "dS" in s else ([o], [s["do"]])
    return [o.detach(), S.detach(), *torch.autograd.grad(outs, list(x.values()), cots)]


def _own_norm(s):
    from delta_feedback_experiment_b200 import layer_norm
    if not s["grad"]:
        return [layer_norm(s["x"], s["weight"], s["bias"], LN_EPS)]
    leaves = [s[n].detach().requires_grad_(True) for n in ("x", "weight", "bias") if s[n] is not None]
    y = layer_norm(*leaves, eps=LN_EPS)
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


def run(state):
    """Rules: output and final state, and in training the gradients of q, k, v, g, beta (and the initial
    state).  Norms: the output, and in training the gradients of x (weight, bias)."""
    if state["kind"] == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------------- the definition
def _exact_rule(q, k, v, g, beta, scale, S0, do, dS, grad):
    """Token by token in fp64 on ``[N, T, H, D]``: output, final state and the gradients of every input.
    Rows of the state are kept every CHUNK tokens and rebuilt inside a chunk on the way back."""
    N, T, H, D = v.shape
    a = g.exp()
    col = lambda t: t[..., None]  # noqa: E731
    S = S0.clone()
    o, kept = torch.empty_like(v), []

    def forward(S, t):
        S = S * col(col(a[:, t]))
        u = col(beta[:, t]) * (v[:, t] - (k[:, t, :, None, :] @ S)[..., 0, :])
        return S + col(k[:, t]) * u[..., None, :]

    for t in range(T):
        if t % CHUNK == 0:
            kept.append(S)
        S = forward(S, t)
        o[:, t] = scale * (q[:, t, :, None, :] @ S)[..., 0, :]
    last = S
    if not grad:
        return o, last, ()
    dq, dk, dv, dg, db = (torch.zeros_like(t) for t in (q, k, v, g, beta))
    dS = torch.zeros_like(last) if dS is None else dS.clone()
    for c in reversed(range(len(kept))):
        states = [kept[c]]
        end = min(T, (c + 1) * CHUNK)
        for t in range(c * CHUNK, end):
            states.append(forward(states[-1], t))
        for t in reversed(range(c * CHUNK, end)):
            before, after = states[t - c * CHUNK], states[t - c * CHUNK + 1]
            qt, kt, dot, at, bt = q[:, t], k[:, t], do[:, t], col(a[:, t]), col(beta[:, t])
            dq[:, t] = scale * (after @ col(dot))[..., 0]
            dS = dS + scale * col(qt) * dot[..., None, :]
            rest = v[:, t] - at * (kt[..., None, :] @ before)[..., 0, :]     # v - a S^T k
            du = (kt[..., None, :] @ dS)[..., 0, :]
            dv[:, t] = bt * du
            db[:, t] = (rest * du).sum(-1)
            dk[:, t] = (dS @ col(bt * rest))[..., 0] - at * (before @ col(bt * du))[..., 0]
            dS = dS - col(kt) * (bt * du)[..., None, :]                      # now of a S_{t-1}
            dg[:, t] = a[:, t] * (dS * before).sum((-1, -2))
            dS = dS * col(at)
    return o, last, (dq, dk, dv, dg, db, dS)


def exact(case, seed):
    """What ``run`` returns, from the definition in 64 bits."""
    s = prepare(case, seed)
    f = lambda n: s[n].double()  # noqa: E731
    if case["kind"] == "norm":
        x = f("x")
        mean, var = x.mean(-1, keepdim=True), x.var(-1, unbiased=False, keepdim=True)
        xh, r = (x - mean) / (var + LN_EPS).sqrt(), 1 / (var + LN_EPS).sqrt()
        affine = s["weight"] is not None
        out = [xh * f("weight") + f("bias") if affine else xh]
        if case["grad"]:
            dy = f("dy")
            h = dy * f("weight") if affine else dy
            out.append(r * (h - h.mean(-1, keepdim=True) - xh * (h * xh).mean(-1, keepdim=True)))
            if affine:
                out += [(dy * xh).sum(0), dy.sum(0)]
        return out
    HK, HV, D = case["HK"], case["HV"], case["D"]
    grad, packed = "do" in s, s["lens"] is not None
    ends = [0]
    for length in s["lens"] or []:
        ends.append(ends[-1] + length)
    pieces = []
    for i in range(len(ends) - 1 if packed else 1):
        part = (lambda t: t[:, ends[i]:ends[i + 1]]) if packed else (lambda t: t)
        one = slice(i, i + 1) if packed else slice(None)
        rows = s["v"].shape[0]
        S0 = f("S0")[one] if s["S0"] is not None else torch.zeros(rows, HV, D, D, dtype=torch.float64, device="cuda")
        o, S, d = _exact_rule(*(part(f(n)).repeat_interleave(HV // HK, 2) for n in ("q", "k")), part(f("v")),
                              part(f("g")), part(f("beta")), s["scale"], S0, part(f("do")) if grad else None,
                              f("dS")[one] if "dS" in s else None, grad)
        if grad:  # heads that share a key: their gradients add up
            d = tuple(t.reshape(*t.shape[:2], HK, HV // HK, D).sum(3) for t in d[:2]) + d[2:]
        pieces.append([o, S, *d])
    out = [torch.cat(parts, 1 if packed and i not in (1, 7) else 0) for i, parts in enumerate(zip(*pieces))]
    return out if s["S0"] is not None or not grad else out[:7]


# ------------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "norm":
        R, N = case["rows"], case["dim"]
        size = 2 if case["dtype"] == "bf16" else 4
        params = 8 * N if case["affine"] else 0
        if not case["grad"]:
            return {"bytes": 2 * R * N * size + params, "flops": 8 * R * N}
        # x, dy in; y, dx out; the parameters in and their gradients out
        return {"bytes": 4 * R * N * size + 2 * params, "flops": 20 * R * N}
    HK, HV, D = case["HK"], case["HV"], case["D"]
    size = 2 if case["dtype"] == "bf16" else 4
    packed = case["kind"] == "packed"
    seqs = len(_lengths(case)) if packed else case["B"]
    tokens = case["total"] if packed else case["B"] * case["T"]
    state = seqs * HV * D * D * 4
    keys, values, scalars = tokens * HK * D * size, tokens * HV * D * size, tokens * HV
    given = case["kind"] == "recurrent" or case["state"]
    read = 2 * keys + values + scalars * (4 + size) + (state if given else 0)
    write = values + state
    # the recurrence itself: two products with the state and one update of it, per token and head
    flops = tokens * HV * 6 * D * D
    if case["kind"] in ("train", "packed"):
        read += values + (state if case["state"] else 0)
        write += 2 * keys + values + scalars * (4 + size) + (state if case["state"] else 0)
        flops *= 3
    return {"bytes": read + write, "flops": flops}
