"""``qk_norm_rotate`` is the dispatcher's operator to whatever looks on: modes, fake tensors, transforms see every call, with a graph
and without one."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from delta_feedback_experiment_b200 import qk_norm_rotate
from test_layer_norm_dispatch_gpu import Seen

pytestmark = pytest.mark.gpu


def inputs(dtype=torch.float32, grad=False):
    gen = torch.Generator().manual_seed(1)
    n = lambda *s: torch.randn(s, generator=gen).cuda()  # noqa: E731
    return (n(2, 5, 4, 32).to(dtype).requires_grad_(grad), n(2, 5, 2, 32).to(dtype), n(32), None, n(16).abs(),
            torch.arange(5, device="cuda"))


@pytest.mark.parametrize("grad", [False, True], ids=["no graph", "graph"])
def test_a_mode_sees_the_call(grad):
    want = qk_norm_rotate(*inputs())
    with Seen() as seen:
        y = qk_norm_rotate(*inputs(grad=grad))
    assert [n for n in seen.names if "delta_feedback" in n] == ["delta_feedback::qk_norm_rotate"]
    assert all(torch.equal(a, b) for a, b in zip(y, want))


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("grad", [False, True], ids=["no graph", "graph"])
def test_fake_tensors_go_through(which, grad):
    """All of the call's tensors are fake ones, or all but the projections (positions and weights that a model keeps)."""
    real = inputs(torch.bfloat16)
    with FakeTensorMode(allow_non_fake_inputs=True):
        x = [None if t is None else torch.empty_like(t, device="cuda") if i < 2 or i != which else t for i, t in enumerate(real)]
        x[0].requires_grad_(grad)
        yq, yk = qk_norm_rotate(*x)
    assert yq.shape == (2, 5, 4, 32) and yk.shape == (2, 5, 2, 32) and yq.dtype == torch.bfloat16 and yq.device.type == "cuda"
    assert yq.requires_grad == grad


def test_a_trace_holds_the_operator():
    from torch.fx.experimental.proxy_tensor import make_fx
    q, k, w, _, freq, at = inputs()
    graph = make_fx(lambda q, k: qk_norm_rotate(q, k, w, None, freq, at))(q, k)
    assert any("qk_norm_rotate" in str(n.target) for n in graph.graph.nodes)
    want = qk_norm_rotate(q, k, w, None, freq, at)
    assert all(torch.equal(a, b) for a, b in zip(graph(q, k), want))


@pytest.mark.parametrize("grad", [False, True], ids=["no graph", "graph"])
def test_a_transform_gets_the_row_by_row_result(grad):
    q, k, w, _, freq, at = inputs(grad=grad)
    y = torch.vmap(lambda a, b: qk_norm_rotate(a[None], b[None], w, None, freq, at))(q, k)
    want = qk_norm_rotate(q, k, w, None, freq, at)
    assert all(torch.equal(a[:, 0], b) for a, b in zip(y, want))


def test_a_transform_of_the_positions_alone():
    q, k, w, _, freq, at = inputs()
    rows = torch.stack((at, at + 100))
    y = torch.vmap(lambda p: qk_norm_rotate(q, k, w, None, freq, p))(rows)
    for i in range(2):
        assert all(torch.equal(a[i], b) for a, b in zip(y, qk_norm_rotate(q, k, w, None, freq, rows[i])))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autocast_changes_nothing(dtype):
    want = qk_norm_rotate(*inputs(dtype))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = qk_norm_rotate(*inputs(dtype))
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(y, want))
