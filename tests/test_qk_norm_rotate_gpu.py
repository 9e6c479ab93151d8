"""qk_norm_rotate against its definition in 64 bits."""

import pytest
import torch

from conftest import assert_close
from oracle.linear_attention_oracle import norm_rotate

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32
HALF_STEP = 2.0 ** -8
# fp32: the mean of up to 256 squares, a root and a quotient, weight, cosine and sine (2^-24 each, an angle to 2^-26 of a
# turn), two products and a sum: some ten roundings of 2^-24, relative to the row's size.
FP32_RTOL = 2.0 ** -19


def make(B, T, HQ, HK, D, R, dtype, seed, first=0, rows=True):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    at = torch.arange(T) + first
    if rows:
        at = at + torch.randint(0, 50, (B, 1), generator=gen)
    return {"q": (1.5 * n(B, T, HQ, D)).to(dtype).cuda(), "k": (0.3 * n(B, T, HK, D)).to(dtype).cuda(),
            "qw": (1 + 0.2 * n(D)).cuda(), "kw": (1 + 0.2 * n(D)).cuda(), "at": at.cuda(),
            "freq": (10000.0 ** (-torch.arange(0, R, 2) / max(R, 1))).float().cuda(),
            "dq": n(B, T, HQ, D).to(dtype).cuda(), "dk": n(B, T, HK, D).to(dtype).cuda()}


def run(d, interleaved=False, eps=1e-6):
    from delta_feedback_experiment_b200 import qk_norm_rotate
    names = [n for n in ("q", "k", "qw", "kw") if d[n] is not None]
    x = {n: d[n].detach().requires_grad_(True) for n in names}
    y = qk_norm_rotate(x["q"], x["k"], x.get("qw"), x.get("kw"), d["freq"], d["at"], eps, interleaved)
    g = torch.autograd.grad(y, list(x.values()), [d["dq"], d["dk"]])
    return {"yq": y[0].detach(), "yk": y[1].detach(), **{"d" + n: t for n, t in zip(names, g)}}


def want(d, interleaved=False, eps=1e-6):
    c = {n: None if t is None else t.detach().cpu() for n, t in d.items()}
    names = [n for n in ("q", "k", "qw", "kw") if d[n] is not None]
    x = {n: c[n].double().requires_grad_(True) for n in names}
    y = [norm_rotate(x[n], x.get(n + "w"), c["freq"], c["at"], eps, interleaved) for n in "qk"]
    g = torch.autograd.grad(y, list(x.values()), [c["dq"].double(), c["dk"].double()])
    return {"yq": y[0].detach(), "yk": y[1].detach(), **{"d" + n: t for n, t in zip(names, g)}}


def compare(got, ref, rows):
    assert set(got) == set(ref)
    for n, t in got.items():
        # a weight's gradient adds up to `rows` fp32 terms of both signs, in a tree of some hundred
        rtol = FP32_RTOL * (4 if n.endswith("w") else 1) + (HALF_STEP if t.dtype == BF16 else 0)
        assert_close(t, ref[n], rtol, n, outlier_frac=0.0)


@pytest.mark.parametrize("B,T,HQ,HK,D,R", [
    (1, 1, 1, 1, 128, 128), (2, 5, 4, 1, 128, 64), (3, 33, 5, 3, 64, 64), (1, 257, 16, 16, 128, 128), (2, 7, 32, 8, 64, 32),
    (1, 19, 3, 2, 256, 256), (2, 11, 2, 2, 96, 96), (1, 13, 1, 7, 90, 42), (2, 9, 3, 1, 2, 2), (1, 8, 2, 2, 254, 100), (1, 6, 8, 1, 32, 16),
    (4, 3, 2, 1, 16, 16), (1, 500, 1, 1, 128, 128), (2, 10, 1, 2, 80, 32), (1, 4, 2, 2, 128, 2), (1, 4, 2, 2, 8, 0)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_values_and_gradients(B, T, HQ, HK, D, R, dtype, interleaved):
    d = make(B, T, HQ, HK, D, R, dtype, 1)
    compare(run(d, interleaved), want(d, interleaved), B * T * HQ)


@pytest.mark.parametrize("B,T,HQ,HK,D,R", [
    (2, 2500, 3, 5, 128, 128),   # a warp has several tokens, one after another
    (1, 500, 36, 40, 128, 64),   # a token's heads go to several warps, not to all the same number
    (1, 1, 41, 7, 64, 64), (3, 1700, 1, 2, 32, 8), (1, 2400, 2, 1, 90, 42)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_work_that_does_not_divide_evenly(B, T, HQ, HK, D, R, dtype):
    d = make(B, T, HQ, HK, D, R, dtype, 9)
    compare(run(d, dtype == FP32), want(d, dtype == FP32), B * T * max(HQ, HK))


@pytest.mark.parametrize("first", [0, 4095, 1_000_003, 2_000_000_000, -777])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_far_positions(first, kind):
    d = make(2, 9, 2, 2, 64, 64, FP32, 2, first=first)
    d["at"] = d["at"].to(kind)
    compare(run(d), want(d), 36)


def test_positions_beyond_32_bits():
    """inv_freq as it is stored is a number of 24 bits, so a position of 2^40 has an angle that 64 bits hold to 2^-20."""
    d = make(1, 4, 1, 1, 32, 32, FP32, 3, first=2 ** 40, rows=False)
    got, ref = run(d), want(d)
    for n in ("yq", "yk"):
        assert_close(got[n], ref[n], 2.0 ** -10, n)


@pytest.mark.parametrize("missing", [("qw",), ("kw",), ("qw", "kw"), ("freq",), ("at",), ("qw", "kw", "freq", "at")])
def test_optional_arguments(missing):
    for dtype in (BF16, FP32):
        d = make(2, 21, 4, 2, 64, 64, dtype, 4, rows=False)
        for n in missing:
            d[n] = None
        compare(run(d), want(d), 168)


def test_slices_of_one_projection_and_odd_starts():
    for dtype in (BF16, FP32):
        for shift in (0, 1):
            d = make(2, 12, 4, 2, 64, 64, dtype, 5)
            row = torch.zeros(2, 12, 8 * 64 + 5, dtype=dtype, device="cuda")
            v = dict(d)
            v["q"] = row[..., shift:shift + 256].unflatten(-1, (4, 64))
            v["k"] = row[..., shift + 256:shift + 384].unflatten(-1, (2, 64))
            v["q"].copy_(d["q"])
            v["k"].copy_(d["k"])
            heads_first = d["dq"].transpose(1, 2).contiguous().transpose(1, 2)
            a, b = run(d), run({**v, "dq": heads_first})
            for n in a:
                if n.endswith("w"):  # (another split of the rows over the lanes: another order of the sum)
                    assert_close(b[n], a[n].double(), 8 * FP32_RTOL, n)
                else:
                    assert_close(b[n], a[n].double(), 2 * FP32_RTOL + (2 * HALF_STEP if dtype == BF16 else 0), n)
            channels_apart = d["q"].transpose(2, 3).contiguous().transpose(2, 3)
            assert torch.equal(run({**d, "q": channels_apart})["yq"], a["yq"])


def test_broadcast_gradient_and_unused_output():
    from delta_feedback_experiment_b200 import qk_norm_rotate
    d = make(2, 5, 2, 2, 32, 32, FP32, 6)
    q, k = d["q"].clone().requires_grad_(True), d["k"].clone().requires_grad_(True)
    yq, yk = qk_norm_rotate(q, k, d["qw"], d["kw"], d["freq"], d["at"])
    yq.sum().backward()
    ref = want({**d, "dq": torch.ones_like(d["q"]), "dk": torch.zeros_like(d["k"])})
    assert_close(q.grad, ref["dq"], FP32_RTOL, "dq")
    assert not k.grad.any()


def test_zero_rows_and_infinities():
    from delta_feedback_experiment_b200 import qk_norm_rotate
    for dtype in (BF16, FP32):
        q = torch.zeros(1, 3, 2, 64, dtype=dtype, device="cuda")
        q[0, 1, 1, 5] = float("nan")
        q[0, 2, 0, 7] = float("inf")
        k = torch.randn(1, 3, 1, 64, device="cuda").to(dtype)
        freq = torch.ones(32, device="cuda")
        yq, yk = qk_norm_rotate(q, k, None, None, freq)
        clean = torch.ones(3, 2, dtype=torch.bool)
        clean[1, 1] = clean[2, 0] = False
        assert not yq[0][clean.cuda()].any() and yq[0, 1, 1].isnan().all() and yk.isfinite().all()
        assert yq[0, 2, 0].isnan().any()


def test_nothing_to_do():
    from delta_feedback_experiment_b200 import qk_norm_rotate
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64), (2, 5, 0, 64)):
        q = torch.randn(shape, device="cuda", requires_grad=True)
        w = torch.ones(64, device="cuda", requires_grad=True)
        yq, yk = qk_norm_rotate(q, q, w, None, torch.ones(32, device="cuda"))
        (yq.sum() + yk.sum()).backward()
        assert yq.shape == q.shape and not w.grad.any()


def test_deterministic_captured_and_compiled():
    from delta_feedback_experiment_b200 import qk_norm_rotate
    d = make(4, 130, 8, 2, 128, 128, BF16, 7)
    a, b = run(d), run(d)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(d)
    e = make(4, 130, 8, 2, 128, 128, BF16, 8)
    for n in d:
        d[n].copy_(e[n])
    graph.replay()
    fresh = run(e)
    for n in out:
        assert torch.equal(out[n], fresh[n]), n

    compiled = torch.compile(lambda q, k, w: qk_norm_rotate(q, k, w, None, e["freq"], e["at"]), fullgraph=True)
    w = e["qw"].clone().requires_grad_(True)
    y = compiled(e["q"], e["k"], w)
    want_y = qk_norm_rotate(e["q"], e["k"], e["qw"], None, e["freq"], e["at"])
    assert torch.equal(y[0], want_y[0]) and torch.equal(y[1], want_y[1])
    y[0].float().sum().backward()
    assert w.grad is not None
    torch.library.opcheck(torch.ops.delta_feedback.qk_norm_rotate.default,
                          (e["q"], e["k"], e["qw"], None, e["freq"], e["at"], 1e-6, False),
                          test_utils=("test_schema", "test_faketensor"))


def test_second_derivative_and_tangents_raise():
    from delta_feedback_experiment_b200 import qk_norm_rotate
    d = make(1, 3, 1, 1, 32, 32, FP32, 9)
    q = d["q"].clone().requires_grad_(True)
    yq, _ = qk_norm_rotate(q, d["k"], d["qw"], d["kw"], d["freq"], d["at"])
    g, = torch.autograd.grad(yq.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(RuntimeError):
        qk_norm_rotate(fwAD.make_dual(d["q"], torch.ones_like(d["q"])), d["k"], None, None, d["freq"])


def test_refusals():
    from delta_feedback_experiment_b200 import qk_norm_rotate
    d = make(2, 6, 2, 2, 64, 64, FP32, 10)

    def refuse(match, **kw):
        x = {**d, **kw}
        with pytest.raises(RuntimeError, match=match):
            qk_norm_rotate(x["q"], x["k"], x["qw"], x["kw"], x["freq"], x["at"])

    refuse("expects q", k=d["k"][:, :5])
    refuse("expects q", k=d["k"][..., :32])
    refuse("even number", q=d["q"][..., :63], k=d["k"][..., :63])
    refuse("weights must be", qw=d["qw"][:32])
    refuse("at most 32 frequencies", freq=torch.ones(33, device="cuda"))
    refuse("int32 or int64", at=d["at"].float())
    refuse("positions must be", at=d["at"][:, :5])
    refuse("bf16 or fp32", q=d["q"].half(), k=d["k"].half())
    refuse("where q is", k=d["k"].bfloat16())
    refuse("no CPU path", k=d["k"].cpu())
    refuse("no gradient of inv_freq", q=d["q"].clone().requires_grad_(True), freq=d["freq"].clone().requires_grad_(True))
