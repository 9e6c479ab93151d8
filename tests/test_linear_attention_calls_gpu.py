"""Calls of linear attention and of the norm and rotation that the documentation allows: offsets that a captured step finds changed, one
output's gradient alone, elements beyond 2^31."""

import ctypes as C

import pytest
import torch

from conftest import assert_close
from delta_feedback_experiment_b200 import _lib
from linear_attention_cases import HALF_STEP, NAMES, SPLIT, attend, make, run_with_grads

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


@pytest.mark.parametrize("T,HV,dtype,D", [(2000, 1, BF16, 128), (2000, 2, BF16, 64), (1100, 160, BF16, 128), (90, 2, FP32, 64)])
@pytest.mark.parametrize("packed", [False, True])
def test_a_prompt_that_writes_over_its_state(T, HV, dtype, D, packed):
    """The C entry point with one state buffer: what two buffers give, up to the order of the segments (fp32, a walk in both: exactly)."""
    lib = _lib.load()
    d = make(1, T, 1, HV, D, dtype, 65, strength=0.002)
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda") if packed else None
    o, S = attend(d, cu=cu)
    a = _lib.LaFwdArgs()
    p, state, out = a.p, d["S0"].clone(), torch.empty_like(d["v"])
    p.n_seqs, p.seq_len, p.total_tokens, p.key_heads, p.value_heads, p.head_dim = 1, T, T, 1, HV, D
    p.dtype, p.scale = (_lib.PKDA_BF16 if dtype == BF16 else _lib.PKDA_F32), D ** -0.5
    p.q, p.k, p.v, p.g = (d[n].data_ptr() for n in NAMES)
    p.cu_seqlens = cu.data_ptr() if packed else None
    p.initial_state = a.final_state = state.data_ptr()
    a.o = out.data_ptr()
    ws = torch.empty(lib.pkda_la_fwd_workspace_bytes(C.byref(p)) + 1, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    assert lib.pkda_la_fwd(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    if not packed:
        assert lib.pkda_last_launch_count() == 1  # (a walk, and not segments side by side, whose first one could find the last one's state)
    torch.cuda.synchronize()
    if dtype == FP32 or HV == 160:
        assert torch.equal(out, o) and torch.equal(state, S)
    else:  # (the operands' parts are cut where the segments are)
        assert_close(state, S, SPLIT, "S")
        assert_close(out, o, SPLIT + 2 * HALF_STEP, "o")


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
