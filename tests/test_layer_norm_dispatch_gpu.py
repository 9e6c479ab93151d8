"""``layer_norm`` is the dispatcher's operator to whatever looks on: modes, fake tensors, transforms see every call, with a graph
and without one."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

from delta_feedback_experiment_b200 import layer_norm

pytestmark = pytest.mark.gpu


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.name())
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("grad", [False, True], ids=["no graph", "graph"])
def test_a_mode_sees_the_call(grad):
    x, w = torch.randn(5, 40, device="cuda"), torch.randn(40, device="cuda")
    want = layer_norm(x, w)
    with Seen() as seen:
        y = layer_norm(x.requires_grad_(grad), w)
    assert seen.names == ["delta_feedback::layer_norm"] and torch.equal(y, want)


@pytest.mark.parametrize("grad", [False, True], ids=["no graph", "graph"])
def test_fake_tensors_go_through(grad):
    with FakeTensorMode():
        x = torch.empty(5, 40, device="cuda", dtype=torch.bfloat16, requires_grad=grad)
        y = layer_norm(x, torch.empty(40, device="cuda"))
    assert y.shape == (5, 40) and y.dtype == torch.bfloat16 and y.device.type == "cuda" and y.requires_grad == grad


def test_a_trace_holds_the_operator():
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(3, 16, device="cuda")
    graph = make_fx(lambda t: layer_norm(t))(x)
    assert any("layer_norm" in str(n.target) for n in graph.graph.nodes)
    assert torch.equal(graph(x), layer_norm(x))


@pytest.mark.parametrize("grad", [False, True], ids=["no graph", "graph"])
def test_a_transform_gets_the_row_by_row_result(grad):
    """vmap has no rule for the operator and calls it row by row."""
    x = torch.randn(4, 3, 16, device="cuda")
    y = torch.vmap(lambda t: layer_norm(t))(x.requires_grad_(grad))
    assert torch.equal(y, layer_norm(x))


def test_autocast_changes_nothing():
    x = torch.randn(3, 16, device="cuda")
    want = layer_norm(x)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(layer_norm(x), want)


def test_forward_mode_raises():
    from torch.autograd import forward_ad
    x = torch.randn(3, 16, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="jvp"):
            layer_norm(forward_ad.make_dual(x, torch.ones_like(x)))
