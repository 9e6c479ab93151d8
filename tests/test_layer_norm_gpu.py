"""Layer norm and its gradients on the GPU against the definition in 64 bits."""

import pytest
import torch

from oracle.delta_rule_oracle import layer_norm_oracle

pytestmark = pytest.mark.gpu
bf16, f32 = torch.bfloat16, torch.float32


def norm(*a, **k):
    from delta_feedback_experiment_b200 import layer_norm
    return layer_norm(*a, **k)


def make(rows, dim, dtype, affine, seed, shift=0.3):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    x, dy = (n(rows, dim) * 1.5 + shift).to(dtype), n(rows, dim).to(dtype)
    w, b = (1 + 0.3 * n(dim), 0.3 * n(dim)) if affine else (None, None)
    return [None if t is None else t.cuda() for t in (x, w, b, dy)]


def run(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = norm(leaves[0], *(leaves[1:] if w is not None else (None, None)), eps=eps)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def want(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().double().cpu().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = layer_norm_oracle(leaves[0], *(leaves[1:] if w is not None else (None, None)), eps=eps)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy.double().cpu())]


def close(got, exp, dtype, rows, where, t=None, eps=1e-5):
    """y and dx: a rounding to the type (half a step: 2^-8 or 2^-24 of the value), and the fp32 arithmetic of a row, 64
    roundings of 2^-24 of what is added up there, which may be more than what is left of it: the mean is off by a part of the
    largest |x|, which reaches y times rstd |w|; dx is rstd (h - mean(h) - xh mean(h xh)), whose three terms are at most
    max|h| times 1, 1 and max|xh|^2, and xh in them is off like y.  dw and db: sums of `rows` terms in an order of at most
    rows / 32 + 64 steps, each off by at most 2^-24 of the sum of the terms' magnitudes, plus rows times xh's own error."""
    half, ulp = (2.0 ** -8 if dtype == bf16 else 2.0 ** -24), 2.0 ** -24
    x, w, b, dy = (None if s is None else s.double().cpu() for s in t)
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w
    c = x - x.mean(-1, keepdim=True)
    rstd = 1 / (c.square().mean(-1, keepdim=True) + eps).sqrt()
    xh, most = c * rstd, lambda s: s.abs().amax(-1, keepdim=True)
    e_xh = 64 * ulp * (rstd * most(x) + most(xh))
    h = dy * w
    e = [e_xh * w.abs() + 64 * ulp * (0 if b is None else b.abs()),
         rstd * most(h) * (64 * ulp * (2 + most(xh) ** 2) + 2 * most(xh) * e_xh),
         (rows / 32 + 64) * ulp * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0),
         (rows / 32 + 64) * ulp * dy.abs().sum(0)]
    for i, (a, want_i) in enumerate(zip(got, exp)):
        a = a.double().cpu()
        assert torch.isfinite(a).all(), where
        bound = (half * want_i.abs() if i < 2 else 0) + e[i] * (1 + half)
        assert ((a - want_i).abs() <= bound).all(), (where, i, ((a - want_i).abs() / (bound + 1e-300)).max().item())


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 8), (9, 33), (17, 64), (4, 255), (64, 256), (7, 257), (33, 512), (130, 513),
          (3, 1000), (1001, 1003), (5, 1024), (20, 2048), (3, 2049), (6, 4096), (2, 4100), (3, 8192), (2, 8200),
          (4, 16384), (2, 16383), (2, 16392), (1, 20001), (3000, 40), (700, 8)]


@pytest.mark.parametrize("dtype", [bf16, f32])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_matches_definition(rows, dim, dtype):
    for affine in (True, False):
        t = make(rows, dim, dtype, affine, seed=rows + dim)
        close(run(*t), want(*t), dtype, rows, (rows, dim, affine), t)


def test_many_rows():
    t = make(20000, 128, bf16, True, seed=1)
    close(run(*t), want(*t), bf16, 20000, "many rows", t)


@pytest.mark.parametrize("dim", [40, 301, 696, 1500, 2600])
@pytest.mark.parametrize("dtype", [bf16, f32])
def test_several_rows_a_turn_and_one_left(dim, dtype):
    t = make(2401, dim, dtype, True, seed=11)
    close(run(*t), want(*t), dtype, 2401, ("odd rows", dim), t)


@pytest.mark.parametrize("dtype", [bf16, f32])
def test_weight_or_bias_alone_and_other_types(dtype):
    x, w, b, dy = make(37, 96, dtype, True, seed=2)
    y = norm(x, w, None)
    close([y], [layer_norm_oracle(x.double().cpu(), w.double().cpu())], dtype, 37, "weight", (x, w, None, dy))
    y = norm(x, None, b)
    close([y], [layer_norm_oracle(x.double().cpu(), None, b.double().cpu())], dtype, 37, "bias", (x, None, b, dy))
    low = [x.requires_grad_(True), w.to(bf16).requires_grad_(True), b.to(bf16).requires_grad_(True)]
    got = torch.autograd.grad(norm(*low), low, dy)
    assert got[1].dtype == bf16 and got[2].dtype == bf16
    only = w.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(norm(x.detach(), only), only, dy)
    full = run(x.detach(), w, b, dy)
    assert torch.equal(dw, full[2])


def test_rows_far_from_zero():
    """The variance is that of the centred values: a mean a thousand times the spread costs digits of x, not of the sum."""
    x, w, b, dy = make(10, 300, f32, True, seed=3, shift=1000.0)
    got, exp = run(x, w, b, dy), want(x, w, b, dy)
    # x itself is given; the mean is off by at most 32 x 2^-24 x 1000, relative to a spread of 1.5
    assert (got[0].double().cpu() - exp[0]).abs().max() < 32 * 2.0 ** -24 * 1000 / 1.5 * 2


def test_constant_rows_infinities_and_nan():
    x, w, b, dy = make(6, 40, f32, True, seed=4)
    x[0] = 3.0
    x[2, 5], x[3, 6] = float("nan"), float("inf")
    got, clean = run(x, w, b, dy), [0, 1, 4, 5]
    exp = want(x[clean], w, b, dy[clean])
    close([got[0][clean], got[1][clean]], exp[:2], f32, 6, "clean rows", (x[clean], w, b, dy[clean]))
    assert torch.isnan(got[0][2]).all() and torch.isnan(got[0][3]).any()


@pytest.mark.parametrize("dtype", [bf16, f32])
def test_strides_and_alignment(dtype):
    x, w, b, dy = make(24, 128, dtype, True, seed=5)
    ref = run(x, w, b, dy)
    flat = torch.zeros(x.numel() + 1, device="cuda", dtype=dtype)
    flat[1:] = x.flatten()
    odd = flat[1:].view_as(x)
    got = run(odd, w, b, dy)
    close(got, want(x, w, b, dy), dtype, 24, "off the grid", (x, w, b, dy))
    pad = torch.zeros(24, 200, device="cuda", dtype=dtype)
    pad[:, 10:138] = x
    got = run(pad[:, 10:138], w, b, dy.t().contiguous().t())
    assert all(torch.equal(a, e) for a, e in zip(got, ref))
    y = norm(x.reshape(2, 3, 4, 128), w, b)
    assert y.shape == (2, 3, 4, 128) and torch.equal(y.reshape(24, 128), ref[0])


def test_repeats_graph_streams():
    x, w, b, dy = make(4000, 640, bf16, True, seed=6)
    ref = run(x, w, b, dy)
    assert all(torch.equal(a, e) for a, e in zip(run(x, w, b, dy), ref))
    with torch.cuda.stream(torch.cuda.Stream()) as _:
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        other = run(x, w, b, dy)
        torch.cuda.current_stream().synchronize()
    assert all(torch.equal(a, e) for a, e in zip(other, ref))
    hx, hdy = torch.zeros_like(x), torch.zeros_like(dy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(hx, w, b, hdy)
    hx.copy_(x)
    hdy.copy_(dy)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(out, ref))


def test_empty():
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y = norm(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert y.shape == (0, 16) and dx.shape == (0, 16) and (dw == 0).all()


def test_compiles_to_one_graph():
    x, w, b, dy = make(10, 64, bf16, True, seed=7)
    ref = run(x, w, b, dy)
    f = torch.compile(lambda x, w, b: norm(x, w, b) * 2, fullgraph=True, backend="aot_eager")
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = f(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y.detach(), ref[0] * 2)
    # twice the cotangent is twice every sum, exactly
    assert all(torch.equal(a, e * 2) for a, e in zip(grads, ref[1:]))


def test_second_derivative_is_refused():
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad(norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(dx.sum(), x)
