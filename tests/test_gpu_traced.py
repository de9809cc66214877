"""The loss in recorded graphs (make_fx, torch.jit.trace) and under dispatch
modes.  A graph holds the operator and gives, for other inputs than those that
it was recorded with, what the eager call gives, bit for bit: both run the same
kernels on the same operands."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from luma_amd import linear_cross_entropy

pytestmark = pytest.mark.gpu

FORWARD = torch.ops.luma_amd.linear_cross_entropy.default
BACKWARD = torch.ops.luma_amd.linear_cross_entropy_backward.default


def _inputs(seed, n=100, h=64, v=300, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((4, n // 4, h), generator=g, device="cuda").to(dtype)
    w = (torch.randn((v, h), generator=g, device="cuda") * 0.2).to(dtype)
    t = torch.randint(0, v, (4, n // 4), generator=g, device="cuda")
    return x.requires_grad_(), w.requires_grad_(), t


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_make_fx(reduction):
    def f(x, w, t):
        loss = linear_cross_entropy(x, w, t, -100, reduction)
        return (loss, *torch.autograd.grad(loss.sum(), (x, w)))

    graph = make_fx(f)(*_inputs(0))
    targets = [node.target for node in graph.graph.nodes]
    assert FORWARD in targets and BACKWARD in targets
    for seed in (1, 2):
        inputs = _inputs(seed)
        got, want = graph(*inputs), f(*inputs)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_make_fx_before_dispatch(reduction):
    """The graph is one of operators that autograd has yet to see.  (Gradients taken
    inside such a graph use what the recorded forward saved, of any operator.)"""
    def f(x, w, t):
        return linear_cross_entropy(x, w, t, -100, reduction)

    graph = make_fx(f, pre_dispatch=True)(*_inputs(0))
    assert FORWARD in [node.target for node in graph.graph.nodes]
    for seed in (1, 2):
        inputs = _inputs(seed)
        got, want = graph(*inputs), f(*inputs)
        assert torch.equal(got, want)
        for p, q in zip(torch.autograd.grad(got.sum(), inputs[:2]),
                        torch.autograd.grad(want.sum(), inputs[:2])):
            assert torch.equal(p, q)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_jit_trace(reduction):
    def f(x, w, t):
        return linear_cross_entropy(x, w, t, -100, reduction)

    graph = torch.jit.trace(f, _inputs(0))
    assert "luma_amd::linear_cross_entropy" in str(graph.graph)
    for seed in (1, 2):
        inputs = _inputs(seed)
        got, want = graph(*inputs), f(*inputs)
        assert torch.equal(got, want)
        for p, q in zip(torch.autograd.grad(got.sum(), inputs[:2]),
                        torch.autograd.grad(want.sum(), inputs[:2])):
            assert torch.equal(p, q)


def test_dispatch_modes_see_both_directions():
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func)
            return func(*args, **(kwargs or {}))

    x, w, t = _inputs(3)
    want_loss = linear_cross_entropy(x, w, t)
    want = torch.autograd.grad(want_loss, (x, w))
    with Mode():
        loss = linear_cross_entropy(x, w, t)
        got = torch.autograd.grad(loss, (x, w))
    assert FORWARD in seen and BACKWARD in seen
    assert torch.equal(loss, want_loss) and all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("pre_dispatch", [False, True])
@pytest.mark.parametrize("only", ["both", "hidden", "weight"])
def test_make_fx_of_the_backward_alone(only, pre_dispatch):
    """The forward ran before the tracer began."""
    x, w, t = _inputs(4)
    loss = linear_cross_entropy(x, w, t, -100, "none")
    wanted = {"both": (x, w), "hidden": (x,), "weight": (w,)}[only]

    def f(g):
        return torch.autograd.grad(loss, wanted, g, retain_graph=True)

    graph = make_fx(f, pre_dispatch=pre_dispatch)(torch.ones_like(loss))
    assert BACKWARD in [node.target for node in graph.graph.nodes]
    for seed in (5, 6):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        g = torch.rand(loss.shape, generator=gen, device="cuda")
        got, want = graph(g), f(g)
        assert len(got) == len(want) and all(torch.equal(p, q) for p, q in zip(got, want))
