"""Linear attention with a decay for each head (chunked and recurrent) and the norm and rotation of
queries and keys in front of it: what is timed, and what it must return.

A case is one call a host makes: a cached decoding step, the prefill of a prompt, the forward +
backward of a training step (dense or packed), or the norm and rotation of one layer's queries and
keys.  ``listed()`` names representative cases, ``draw()`` gives more of the same ranges.

Linear attention, per value head with state ``S [K, V]`` and key head ``h // (HV / HK)``:

    S_t = a_t S_{t-1} + k_t v_t^T,   a_t = exp(g_t),   o_t = scale S_t^T q_t,

``g`` a number a token and head (``[B, T, HV]``) or one a head (``[HV]``).  Norm and rotation, per
row ``x`` of a head, with pairs ``(x_j, x_{j + R/2})`` (or ``(x_{2j}, x_{2j+1})``) of its first ``R`` channels:

    n = x / sqrt(mean(x^2) + eps) * w,   y = n rotated in each pair by position * inv_freq_j.

``run`` computes them in plain torch, 64 tokens at a time in 32 bits, or calls the framework's
operators; ``exact`` goes token by token in 64 bits with the reverse recurrence written out.
"""

from __future__ import annotations

import math
import random

import torch

own = False

CHUNK = 64
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # One user, one token: the latency of a cached decoding step of a small layer.
        {"name": "attend-decode-1", "kind": "recurrent", "B": 1, "T": 1, "HK": 8, "HV": 8, "D": 128, "dtype": "bf16",
         "dist": "production"},
        # 256 users, 32 heads with shared keys: 512 MB of state read and written.
        {"name": "attend-decode-256", "kind": "recurrent", "B": 256, "T": 1, "HK": 16, "HV": 32, "D": 128,
         "dtype": "bf16", "dist": "production"},
        # A few tokens appended to cached rows (a short prompt, a speculative block).
        {"name": "attend-append-48", "kind": "recurrent", "B": 4, "T": 48, "HK": 16, "HV": 16, "D": 128,
         "dtype": "bf16", "dist": "production"},
        # One long prompt of odd length, a fixed decay for each head: forward only, the final state is kept.
        {"name": "attend-prefill-8191", "kind": "prefill", "B": 1, "T": 8191, "HK": 16, "HV": 16, "D": 128,
         "dtype": "bf16", "dist": "heads", "state": False},
        # The headline training shape.
        {"name": "attend-train", "kind": "train", "B": 8, "T": 4096, "HK": 16, "HV": 16, "D": 128, "dtype": "bf16",
         "dist": "unit", "state": False},
        # Value heads that share key heads, states in and out, a ragged length.
        {"name": "attend-train-shared", "kind": "train", "B": 2, "T": 2047, "HK": 4, "HV": 12, "D": 128,
         "dtype": "bf16", "dist": "production", "state": True},
        # Documents of 17 to 4,096 tokens packed to one row.
        {"name": "attend-packed", "kind": "packed", "total": 32768, "lo": 17, "hi": 4096, "cut": 7, "HK": 8, "HV": 16,
         "D": 128, "dtype": "bf16", "dist": "production", "state": True},
        # The fp32 configuration, heads of 64 channels, a decay a head that is learned.
        {"name": "attend-exact", "kind": "train", "B": 2, "T": 512, "HK": 4, "HV": 4, "D": 64, "dtype": "fp32",
         "dist": "heads", "state": True},
        # Queries and keys of a training step, forward and backward with both weights.
        {"name": "rotate-train", "kind": "rotate", "B": 8, "T": 4096, "HQ": 16, "HK": 16, "D": 128, "R": 128,
         "dtype": "bf16", "interleaved": False, "affine": True, "packed": False, "first": 0, "grad": True},
        # Slices of one packed projection of a long prompt, few key heads, half of the channels rotated, forward only.
        {"name": "rotate-prefill-8191", "kind": "rotate", "B": 1, "T": 8191, "HQ": 32, "HK": 4, "D": 64, "R": 32,
         "dtype": "bf16", "interleaved": False, "affine": True, "packed": True, "first": 0, "grad": False},
        # Odd heads and widths in fp32, neighbouring channels as pairs.
        {"name": "rotate-odd", "kind": "rotate", "B": 3, "T": 333, "HQ": 5, "HK": 3, "D": 90, "R": 42,
         "dtype": "fp32", "interleaved": True, "affine": True, "packed": True, "first": 1000, "grad": True},
        # One token of each of 64 users, far into their contexts.
        {"name": "rotate-decode", "kind": "rotate", "B": 64, "T": 1, "HQ": 16, "HK": 16, "D": 128, "R": 128,
         "dtype": "bf16", "interleaved": False, "affine": True, "packed": True, "first": 1000000, "grad": False},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_UNITS = 8 * 4096 * 16       # (token, value head) pairs of a drawn case, at most
HEADS = ((1, 1), (2, 2), (4, 4), (8, 8), (16, 16), (2, 8), (4, 12), (8, 16), (16, 32))


def draw(rng: random.Random):
    kind = rng.choice(("recurrent", "recurrent", "prefill", "train", "train", "packed", "rotate", "rotate", "rotate"))
    if kind == "rotate":
        D = rng.choice((64, 128, 128, 128, 256, 96, 80, 32, 2 * rng.randint(4, 128)))
        R = rng.choice((D, D, D, D // 4 * 2, 2 * rng.randint(1, D // 2)))
        HQ = rng.choice((1, 4, 5, 16, 32))
        HK = rng.choice((HQ, 1, max(1, HQ // 4)))
        B = rng.choice((1, 1, 2, 8, 64))
        most = 8 * 4096 * 32 * 128 // ((HQ + HK) * D * B)
        return {"kind": kind, "B": B, "T": 1 if rng.random() < 0.2 else _log(rng, 1, max(1, min(16384, most))),
                "HQ": HQ, "HK": HK, "D": D, "R": R, "dtype": rng.choice(("bf16", "bf16", "fp32")),
                "interleaved": rng.random() < 0.3, "affine": rng.random() < 0.8, "packed": rng.random() < 0.5,
                "first": rng.choice((0, 0, 77, 123456, 2000000)), "grad": rng.random() < 0.6}
    HK, HV = rng.choice(HEADS)
    dtype, D = rng.choice((("bf16", 128), ("bf16", 128), ("bf16", 128), ("bf16", 64), ("fp32", 64), ("fp32", 128),
                           ("fp32", 32)))
    c = {"kind": kind, "HK": HK, "HV": HV, "D": D, "dtype": dtype, "dist": rng.choice(("unit", "production", "heads"))}
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
    if case["kind"] == "rotate":
        B, T, HQ, HK, D, R = (case[key] for key in ("B", "T", "HQ", "HK", "D", "R"))
        if case["packed"]:  # the projection's row holds queries, keys and values side by side
            row = (1.5 * n(B, T, (HQ + 2 * HK) * D)).to(dt)
            q = row[..., :HQ * D].unflatten(-1, (HQ, D))
            k = row[..., HQ * D:(HQ + HK) * D].unflatten(-1, (HK, D))
        else:
            q, k = (1.5 * n(B, T, HQ, D)).to(dt), (1.5 * n(B, T, HK, D)).to(dt)
        at = torch.arange(T, device="cuda")
        if case["first"]:  # rows that are cached, each up to a place of its own
            at = at + case["first"] + torch.randint(0, 1000, (B, 1), generator=gen, device="cuda")
        s = {"kind": "rotate", "q": q, "k": k, "qw": None, "kw": None, "positions": at, "grad": case["grad"],
             "inv_freq": (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).float().cuda(),
             "interleaved": case["interleaved"]}
        if case["affine"]:
            s["qw"], s["kw"] = 1 + 0.2 * n(D), 1 + 0.2 * n(D)
        if case["grad"]:
            s["dyq"], s["dyk"] = n(B, T, HQ, D).to(dt), n(B, T, HK, D).to(dt)
        return s
    packed = case["kind"] == "packed"
    lens = _lengths(case) if packed else None
    B, T = (1, case["total"]) if packed else (case["B"], case["T"])
    HK, HV, D = case["HK"], case["HV"], case["D"]
    N = len(lens) if packed else B
    silu = torch.nn.functional.silu
    unit = case["dist"] == "unit"
    norm = lambda t: t / t.square().sum(-1, keepdim=True).add(1e-6).sqrt()  # noqa: E731
    # keys and queries as a norm leaves them, behind a short convolution with SiLU or evenly spread
    q, k = (norm(n(B, T, HK, D) if unit else silu(n(B, T, HK, D))).to(dt) for _ in range(2))
    v = (n(B, T, HV, D) if unit else silu(n(B, T, HV, D))).to(dt)
    if unit:
        g = -torch.nn.functional.softplus(n(B, T, HV))
    elif case["dist"] == "heads":  # windows from a few tokens to thousands, one for each head
        g = -torch.exp2(-8.0 * (torch.arange(HV, device="cuda") + u(0.5, 1.5, HV)) / HV)
    else:  # exp(A_log) ~ U(1, 16) and steps of 1e-3 to 1e-1, as such layers are initialised
        step = u(math.log(1e-3), math.log(1e-1), HV).exp()
        bias = step + torch.log(-torch.expm1(-step))
        g = -u(1.0, 16.0, HV) * torch.nn.functional.softplus(0.5 * n(B, T, HV) + bias)
    s = {"kind": case["kind"], "q": q, "k": k, "v": v, "g": g, "scale": D ** -0.5, "S0": None, "lens": lens,
         "cu": None}
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
def _plain_step(q, k, v, g, scale, S):
    """One token: [B, HV, D] rows on S [B, HV, D, D], everything fp32."""
    S = S * g.exp()[..., None, None] + k[..., None] * v[..., None, :]
    return scale * (S * q[..., None]).sum(-2), S


def _plain_attend(q, k, v, g, scale, S):
    """``[N, T, H, D]`` fp32 rows (keys and queries repeated to the value heads), state or None ->
    output and final state, a chunk of 64 tokens at a time."""
    N, T, H, D = v.shape
    NC = -(-T // CHUNK)
    pad = NC * CHUNK - T

    def cut(t):  # [N, T, H, ...] -> [N, H, NC, 64, ...]; added rows are zero and leave the state alone
        if pad:
            t = torch.cat((t, t.new_zeros(N, pad, *t.shape[2:])), 1)
        return t.reshape(N, NC, CHUNK, *t.shape[2:]).movedim(3, 1)

    q, k, v, g = (cut(t) for t in (q, k, v, g))
    G = g.double().cumsum(-1)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=v.device).tril()
    decay = (G[..., :, None] - G[..., None, :]).float().masked_fill(~low, -math.inf).exp()
    P = scale * (q @ k.transpose(-1, -2)) * decay
    kd = k * (G[..., -1:] - G).float().exp()[..., None]
    qd = scale * q * G.float().exp()[..., None]
    whole = G[..., -1].float().exp()
    inside, writes = P @ v, kd.transpose(-1, -2) @ v
    S = v.new_zeros(N, H, D, D) if S is None else S
    o = []
    for c in range(NC):
        o.append(qd[:, :, c] @ S + inside[:, :, c])
        S = S * whole[:, :, c, None, None] + writes[:, :, c]
    return torch.stack(o, 2).movedim(1, 3).reshape(N, NC * CHUNK, H, D)[:, :T], S


def _plain(s):
    dt, HK, HV = s["v"].dtype, s["k"].shape[2], s["v"].shape[2]
    grad = "do" in s
    names = ["q", "k", "v", "g"] + (["S0"] if s["S0"] is not None else [])
    x = {n: s[n].float().requires_grad_(grad) for n in names}
    wide = {n: x[n].repeat_interleave(HV // HK, 2) for n in ("q", "k")}
    rows = [wide["q"], wide["k"], x["v"], x["g"].expand(s["v"].shape[:3])]
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
            o, S = _plain_attend(*rows, s["scale"], S0)
            o = o[real][None]
        elif s["v"].shape[1] == 1:
            o, S = _plain_step(*(t[:, 0] for t in rows), s["scale"], S0 if S0 is not None else 0.0)
            o = o[:, None]
        else:
            o, S = _plain_attend(*rows, s["scale"], S0)
    if not grad:
        return [o.to(dt), S]
    outs, cots = ([o, S], [s["do"].float(), s["dS"]]) if "dS" in s else ([o], [s["do"].float()])
    grads = torch.autograd.grad(outs, list(x.values()), cots)
    return [o.detach().to(dt), S.detach()] + [d.to(s[n].dtype) for n, d in zip(names, grads)]


def _plain_rotate(s):
    grad, dt = s["grad"], s["q"].dtype
    angle = s["positions"].double()[..., None, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    half = s["inv_freq"].numel()
    x = {n: s[n].float().requires_grad_(grad) for n in ("q", "k", "qw", "kw") if s[n] is not None}

    def one(t, w):
        t = t * (t.square().mean(-1, keepdim=True) + EPS).rsqrt()
        if w is not None:
            t = t * w
        r, rest = t[..., :2 * half], t[..., 2 * half:]
        a, b = (r[..., 0::2], r[..., 1::2]) if s["interleaved"] else (r[..., :half], r[..., half:])
        a, b = a * cos - b * sin, b * cos + a * sin
        r = torch.stack((a, b), -1).flatten(-2) if s["interleaved"] else torch.cat((a, b), -1)
        return torch.cat((r, rest), -1)

    with torch.set_grad_enabled(grad):
        y = [one(x["q"], x.get("qw")), one(x["k"], x.get("kw"))]
    if not grad:
        return [t.to(dt) for t in y]
    d = torch.autograd.grad(y, list(x.values()), [s["dyq"].float(), s["dyk"].float()])
    return [t.detach().to(dt) for t in y] + [t.to(s[n].dtype) for n, t in zip(x, d)]


# ------------------------------------------------------------- the framework's calls
def _own(s):
    from delta_feedback_experiment_b200 import chunk_linear_attention, fused_recurrent_linear_attention
    if s["kind"] == "recurrent":
        o, S = fused_recurrent_linear_attention(s["q"], s["k"], s["v"], s["g"], scale=s["scale"],
                                                initial_state=s["S0"], output_final_state=True)
        return [o, S]
    grad = "do" in s
    names = ["q", "k", "v", "g"] + (["S0"] if s["S0"] is not None else [])
    x = {n: s[n].detach().requires_grad_(grad) for n in names}
    o, S = chunk_linear_attention(x["q"], x["k"], x["v"], x["g"], scale=s["scale"], initial_state=x.get("S0"),
                                  output_final_state=True, cu_seqlens=s["cu"])
    if not grad:
        return [o, S]
    outs, cots = ([o, S], [s["do"], s["dS"]]) if "dS" in s else ([o], [s["do"]])
    return [o.detach(), S.detach(), *torch.autograd.grad(outs, list(x.values()), cots)]


def _own_rotate(s):
    from delta_feedback_experiment_b200 import qk_norm_rotate
    names = [n for n in ("q", "k", "qw", "kw") if s[n] is not None]
    x = {n: s[n].detach().requires_grad_(s["grad"]) for n in names}
    y = qk_norm_rotate(x["q"], x["k"], x.get("qw"), x.get("kw"), s["inv_freq"], s["positions"], eps=EPS,
                       interleaved=s["interleaved"])
    if not s["grad"]:
        return list(y)
    return [t.detach() for t in y] + list(torch.autograd.grad(y, list(x.values()), [s["dyq"], s["dyk"]]))


def run(state):
    """Attention: output and final state, and in training the gradients of q, k, v, g (and the initial state).
    Norm and rotation: both outputs, and in training the gradients of q, k (and of both weights)."""
    if state["kind"] == "rotate":
        return _own_rotate(state) if own else _plain_rotate(state)
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------------- the definition
def _exact_attend(q, k, v, g, scale, S0, do, dS, grad):
    """Token by token in fp64 on ``[N, T, H, D]``: output, final state and the gradients of every input.
    Rows of the state are kept every CHUNK tokens and rebuilt inside a chunk on the way back."""
    T = v.shape[1]
    a = g.exp()
    col = lambda t: t[..., None]  # noqa: E731
    S = S0.clone()
    o, kept = torch.empty_like(v), []

    def forward(S, t):
        return S * col(col(a[:, t])) + col(k[:, t]) * v[:, t, :, None, :]

    for t in range(T):
        if t % CHUNK == 0:
            kept.append(S)
        S = forward(S, t)
        o[:, t] = scale * (q[:, t, :, None, :] @ S)[..., 0, :]
    last = S
    if not grad:
        return o, last, ()
    dq, dk, dv, dg = (torch.zeros_like(t) for t in (q, k, v, g))
    dS = torch.zeros_like(last) if dS is None else dS.clone()
    for c in reversed(range(len(kept))):
        states = [kept[c]]
        end = min(T, (c + 1) * CHUNK)
        for t in range(c * CHUNK, end):
            states.append(forward(states[-1], t))
        for t in reversed(range(c * CHUNK, end)):
            before, after = states[t - c * CHUNK], states[t - c * CHUNK + 1]
            dot = do[:, t]
            dq[:, t] = scale * (after @ col(dot))[..., 0]
            dS = dS + scale * col(q[:, t]) * dot[..., None, :]
            dk[:, t] = (dS @ col(v[:, t]))[..., 0]
            dv[:, t] = (k[:, t, :, None, :] @ dS)[..., 0, :]
            dg[:, t] = a[:, t] * (dS * before).sum((-1, -2))
            dS = dS * col(col(a[:, t]))
    return o, last, (dq, dk, dv, dg, dS)


def _exact_rotate(case, s):
    R, D = case["R"], case["D"]
    pos = s["positions"].double()
    freq = s["inv_freq"].double()
    first = torch.arange(R // 2, device="cuda") * (2 if s["interleaved"] else 1)
    second = first + (1 if s["interleaved"] else R // 2)
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos[..., None] * freq)[..., None, :]

    def turn(t, z):  # pairs as complex numbers
        t = t.clone()
        c = torch.complex(t[..., first], t[..., second]) * z
        t[..., first], t[..., second] = c.real, c.imag
        return t

    ys, dxs, dws = [], [], []
    for name in ("q", "k"):
        x = s[name].double()
        w = s[name + "w"].double() if s[name + "w"] is not None else torch.ones(D, dtype=torch.float64, device="cuda")
        r = (x.pow(2).sum(-1, keepdim=True) / D + EPS).pow(-0.5)
        ys.append(turn(x * r * w, z))
        if case["grad"]:
            h = turn(s["dy" + name].double(), z.conj())
            dws.append((h * x * r).sum((0, 1, 2)))
            h = h * w
            dxs.append(r * h - x * r.pow(3) * (h * x).sum(-1, keepdim=True) / D)
    return ys + dxs + (dws if case["affine"] else [])


def exact(case, seed):
    """What ``run`` returns, from the definition in 64 bits."""
    s = prepare(case, seed)
    if case["kind"] == "rotate":
        return _exact_rotate(case, s)
    f = lambda n: s[n].double()  # noqa: E731
    HK, HV, D = case["HK"], case["HV"], case["D"]
    grad, packed = "do" in s, s["lens"] is not None
    ends = [0]
    for length in s["lens"] or []:
        ends.append(ends[-1] + length)
    g = f("g").expand(s["v"].shape[:3]).contiguous()
    pieces = []
    for i in range(len(ends) - 1 if packed else 1):
        part = (lambda t: t[:, ends[i]:ends[i + 1]]) if packed else (lambda t: t)
        one = slice(i, i + 1) if packed else slice(None)
        rows = s["v"].shape[0]
        S0 = f("S0")[one] if s["S0"] is not None else torch.zeros(rows, HV, D, D, dtype=torch.float64, device="cuda")
        o, S, d = _exact_attend(*(part(f(n)).repeat_interleave(HV // HK, 2) for n in ("q", "k")), part(f("v")),
                                part(g), s["scale"], S0, part(f("do")) if grad else None,
                                f("dS")[one] if "dS" in s else None, grad)
        if grad:  # heads that share a key: their gradients add up
            d = tuple(t.reshape(*t.shape[:2], HK, HV // HK, D).sum(3) for t in d[:2]) + d[2:]
        pieces.append([o, S, *d])
    out = [torch.cat(parts, 1 if packed and i not in (1, 6) else 0) for i, parts in enumerate(zip(*pieces))]
    if grad and s["g"].dim() == 1:  # one decay a head: its gradient is the sum over the tokens
        out[5] = out[5].sum((0, 1))
    return out if s["S0"] is not None or not grad else out[:6]


# ------------------------------------------------------------------------------- work
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "rotate":
        tokens = case["B"] * case["T"]
        rows = tokens * (case["HQ"] + case["HK"])
        x, small = rows * case["D"] * size, tokens * 8 + 2 * case["R"] + (8 * case["D"] if case["affine"] else 0)
        if not case["grad"]:
            return {"bytes": 2 * x + small, "flops": rows * (4 * case["D"] + 3 * case["R"])}
        # q, k, their outputs' gradients in; the outputs and the gradients out
        return {"bytes": 4 * x + small + (8 * case["D"] if case["affine"] else 0),
                "flops": rows * (14 * case["D"] + 6 * case["R"])}
    HK, HV, D = case["HK"], case["HV"], case["D"]
    packed = case["kind"] == "packed"
    seqs = len(_lengths(case)) if packed else case["B"]
    tokens = case["total"] if packed else case["B"] * case["T"]
    state = seqs * HV * D * D * 4
    keys, values = tokens * HK * D * size, tokens * HV * D * size
    gates = HV * 4 if case["dist"] == "heads" else tokens * HV * 4
    given = case["kind"] == "recurrent" or case["state"]
    read = 2 * keys + values + gates + (state if given else 0)
    write = values + state
    # the recurrence itself: one update of the state and one product with it, per token and head
    flops = tokens * HV * 4 * D * D
    if case["kind"] in ("train", "packed"):
        read += values + (state if case["state"] else 0)
        write += 2 * keys + values + gates + (state if case["state"] else 0)
        flops *= 3
    return {"bytes": read + write, "flops": flops}
