"""Calls of linear attention and of the norm and rotation that the documentation allows: offsets that a captured step finds changed, one
output's gradient alone, elements beyond 2^31."""

import pytest
import torch

from linear_attention_cases import NAMES, attend, make, run_with_grads

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,D,HV,lens", [
    (BF16, 128, 1, ((1300, 900), (0, 2200), (1, 1000))), (BF16, 128, 40, ((700, 1, 300), (64, 800, 0), (5, 5, 5))),
    (BF16, 64, 2, ((300, 20, 400), (0, 0, 720), (65, 64, 63))), (FP32, 32, 2, ((100, 20, 50), (0, 0, 170), (1, 2, 3)))])
def test_a_captured_step_takes_new_offsets(dtype, D, HV, lens):
    total = sum(lens[0]) + 9
    cuts = [torch.tensor([3] + [3 + sum(x[:i + 1]) for i in range(len(x))], dtype=torch.int32, device="cuda") for x in lens]
    d = make(1, total, 1, HV, D, dtype, 61, N=len(lens[0]), strength=0.02)
    cu = cuts[0].clone()
    leaves = {n: d[n].detach().clone().requires_grad_(True) for n in (*NAMES, "S0")}

    def step():
        o, S = attend({**d, **leaves}, cu=cu)
        return [o, S, *torch.autograd.grad([o, S], list(leaves.values()), [d["do"], d["dS"]])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for c in (*cuts, cuts[0]):
        cu.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        want = run_with_grads(d, cu=c)
        for t, n in zip(out, ("o", "S", "dq", "dk", "dv", "dg", "dS0")):
            assert torch.equal(t, want[n]), n


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (FP32, 64)])
def test_the_gradient_of_one_output_alone(dtype, D):
    d = make(2, 200, 1, 2, D, dtype, 62)
    zero = {"o": torch.zeros_like(d["do"]), "S": torch.zeros_like(d["dS"])}
    for which in ("o", "S"):
        leaves = {n: d[n].detach().clone().requires_grad_(True) for n in (*NAMES, "S0")}
        o, S = attend({**d, **leaves})
        got = torch.autograd.grad(o if which == "o" else S, list(leaves.values()), d["do"] if which == "o" else d["dS"])
        both = run_with_grads({**d, "dS": zero["S"]} if which == "o" else {**d, "do": zero["o"]})
        for n, t in zip(leaves, got):
            assert torch.equal(t, both["d" + n]), (which, n)


def test_elements_beyond_32_bits():
    """The last of two sequences lies behind element 2^31 of every activation, and comes out as it does alone."""
    H, D, last = 64, 128, 200
    T = 2 ** 31 // (H * D) + 1000
    small = make(1, last, H, H, D, BF16, 63, N=1, strength=0.1)
    d = {n: torch.zeros((1, T, *small[n].shape[2:]), dtype=small[n].dtype, device="cuda") for n in ("q", "k", "v", "g", "do")}
    for n in d:
        d[n][:, T - last:] = small[n]
    for n in ("S0", "dS"):
        d[n] = torch.cat((torch.zeros_like(small[n]), small[n]))
    got, want = run_with_grads(d, cu=torch.tensor([0, T - last, T], dtype=torch.int32, device="cuda")), run_with_grads(small)
    for n in ("o", "dq", "dk", "dv", "dg"):
        assert torch.equal(got[n][:, T - last:], want[n]), n
        assert not got[n][:, :T - last].any(), n
    for n in ("S", "dS0"):
        assert torch.equal(got[n][1:], want[n]) and not got[n][0].any(), n


@pytest.mark.parametrize("batch", [1, 2])
def test_rotation_of_elements_beyond_32_bits(batch):
    from delta_feedback_experiment_b200 import qk_norm_rotate
    H, D, last = 64, 128, 50
    T = (2 ** 31 // (H * D) + 500) // batch
    gen = torch.Generator().manual_seed(64)
    n = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    small = [n(1, last, H, D).bfloat16().cuda() for _ in range(2)]
    q, k, dy = (torch.zeros(batch, T, H, D, dtype=BF16, device="cuda") for _ in range(3))
    w, freq = n(D).cuda(), n(D // 2).abs().cuda()
    q[-1, T - last:], k[-1, T - last:] = small[0], small[0]
    dy[-1, T - last:] = small[1]
    at = torch.arange(T, device="cuda")
    results = []
    for x, y, c, p in ((q, k, dy, at), (small[0], small[0], small[1], at[T - last:])):
        x, y = x.detach().requires_grad_(True), y.detach().requires_grad_(True)
        out = qk_norm_rotate(x, y, w, w, freq, p)
        results.append([t.detach() for t in out] + list(torch.autograd.grad(out, (x, y), (c, c))))
    for a, b in zip(*results):
        assert torch.equal(a[-1:, T - last:], b)
        assert not a[-1, :T - last].any() and not a[:-1].any()
