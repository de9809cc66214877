"""add_layer_norm whose y a program does not use: the sum's gradients alone."""

import math

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import residual_util
from luma_amd import _lib as L
from luma_amd import add_layer_norm, dropout

pytestmark = pytest.mark.gpu

TYPES = [(d, d) for d in (torch.float32, torch.bfloat16, torch.float16)] + [
    (torch.float32, torch.bfloat16), (torch.float32, torch.float16)]
N, H = 20, 66


@pytest.fixture(params=["the host module", "operators"])
def path(request, monkeypatch):
    if request.param == "operators":
        monkeypatch.setattr(L, "host_calls", lambda: None)


def _inputs(stream, branch):
    """Rows that a norm has no finite gradient for among them: an infinity, a NaN, and
    (with eps = 0) a constant row."""
    g = torch.Generator(device="cuda").manual_seed(5)

    def randn(shape, dtype):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    x, res, d = randn((N, H), branch), randn((N, H), stream), randn((N, H), stream)
    res[2, 3], res[5, H - 1], res[7, 0] = math.inf, math.nan, -math.inf
    x[9], res[9] = 0.0, 1.0
    w, b = randn((H,), branch), randn((H,), branch)
    return [t.requires_grad_() for t in (x, res, w, b)], d


@pytest.mark.parametrize("stream,branch", TYPES)
@pytest.mark.parametrize("p", [0.0, 0.5, 1.0])
def test_the_sum_alone(path, p, stream, branch):
    leaves, d = _inputs(stream, branch)
    _, total = add_layer_norm(*leaves, 0.0, p, 3, 4)
    got = torch.autograd.grad(total, leaves, d, retain_graph=True)
    keep = residual_util.kept((N, H), p, 3, 4).cuda()
    # (1 / (1 - p) is 1 or 2 here: one rounding to the branch's type)
    want = torch.where(keep, d.float() * (1.0 / (1.0 - p) if p < 1.0 else 0.0), 0.0).to(branch)
    assert torch.equal(got[1], d) and torch.equal(got[0], want) and got[0].dtype == branch
    for t, leaf in zip(got[2:], leaves[2:]):
        assert t.dtype == leaf.dtype and t.shape == leaf.shape and bool((t == 0).all())
    for i, leaf in enumerate(leaves):               # each alone
        one, = torch.autograd.grad(total, leaf, d, retain_graph=True)
        assert torch.equal(one, got[i])
    # as dropout onto the residual
    y = dropout(leaves[0], p, 3, 4, residual=leaves[1])
    assert all(torch.equal(s, t) for s, t in zip(torch.autograd.grad(y, leaves[:2], d), got))


@pytest.mark.parametrize("p", [0.0, 0.5])
def test_in_recorded_graphs(p):
    """No norm is differentiated there."""
    leaves, d = _inputs(torch.float32, torch.bfloat16)

    def f(d):
        return torch.autograd.grad(add_layer_norm(*leaves, 0.0, p, 3, 4)[1], leaves, d)

    graph = make_fx(f)(torch.ones_like(d))
    assert torch.ops.luma_amd.layer_norm_backward.default not in [n.target for n in graph.graph.nodes]
    assert all(torch.equal(s, t) for s, t in zip(graph(d), f(d)))


@pytest.mark.parametrize("p", [0.0, 0.5])
def test_captured(p):
    leaves, d = _inputs(torch.float32, torch.bfloat16)

    def step():
        return torch.autograd.grad(add_layer_norm(*leaves, 0.0, p, 3, 4)[1], leaves, d)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        d.mul_(2.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))


@pytest.mark.parametrize("p", [0.0, 0.5])
def test_accumulated(p):
    """Into .grad, where the sum's gradient goes to both operands."""
    leaves, d = _inputs(torch.float32, torch.float32)
    kept = d.clone()
    for _ in range(2):
        add_layer_norm(*leaves, 0.0, p, 3, 4)[1].backward(d)
    assert torch.equal(d, kept) and torch.equal(leaves[1].grad, 2 * d)
    keep = residual_util.kept((N, H), p, 3, 4).cuda()
    assert torch.equal(leaves[0].grad, torch.where(keep, d * (2 / (1 - p)), 0.0))
    assert all(bool((leaf.grad == 0).all()) for leaf in leaves[2:])
    x, res = (t.detach().requires_grad_() for t in leaves[:2])
    (add_layer_norm(x, res, p=p, seed=3)[1] * d).backward(torch.ones_like(d))
    assert x.grad.data_ptr() != res.grad.data_ptr() and torch.equal(res.grad, d)


def test_differentiated_again(path):
    leaves, d = _inputs(torch.float32, torch.float32)
    total = add_layer_norm(*leaves, 0.0, 0.5, 3, 4)[1]
    g, = torch.autograd.grad(total, leaves[0], d.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="cannot|does not|no autograd"):
        g.sum().backward()


@pytest.mark.parametrize("where", ["in the step", "after it"])
@pytest.mark.parametrize("compiled", [False, True])
def test_a_seed_written_before_the_backward_is_told(compiled, where):
    """The masks would be others: eager and compiled programs raise."""
    x = torch.ones(4096, device="cuda", requires_grad=True)

    def step(x, seed):
        y = dropout(x, 0.5, seed, 1)
        z = add_layer_norm(y.view(64, 64), y.view(64, 64), p=0.5, seed=seed, call=2)[1]
        if where == "in the step":
            seed.add_(1)
        return z

    seed = torch.tensor(7, device="cuda")
    # (of a step that writes it itself the compiler says so, when it records the backward)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z = (torch.compile(step, fullgraph=True) if compiled else step)(x, seed)
        if where == "after it":
            seed += 1
        z.sum().backward()


@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("stream,branch", [(torch.float32, torch.float32),
                                           (torch.float32, torch.bfloat16)])
def test_the_sum_alone_compiled(stream, branch, p):
    leaves, d = _inputs(stream, branch)

    def f(*leaves):
        return add_layer_norm(*leaves, 0.0, p, 3, 4)[1]

    want = torch.autograd.grad(f(*leaves), leaves, d)
    got = torch.autograd.grad(torch.compile(f, fullgraph=True)(*leaves), leaves, d)
    assert all(torch.equal(s, t) for s, t in zip(got, want))
    got = torch.autograd.grad(torch.compile(lambda *a: f(*a) * 1.0, fullgraph=True)(*leaves), leaves, d)
    assert all(torch.equal(s, t) for s, t in zip(got, want))
