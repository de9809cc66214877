"""The residual stream's operators and the policy loss in recorded graphs
(make_fx, torch.jit.trace, torch.compile) and under dispatch modes: a graph
holds the operators and gives, for other inputs than those that it was recorded
with, what the eager call gives, bit for bit."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from luma_amd import add_layer_norm, dropout, layer_norm, policy_loss

pytestmark = pytest.mark.gpu

OPS = torch.ops.luma_amd


def _norm(x, r, w, b):
    return layer_norm(x, w, b)


def _norm_mixed(x, r, w, b):
    return layer_norm(x, w, b, dtype=torch.bfloat16)


def _add(x, r, w, b):
    y, total = add_layer_norm(x, r, w, b, p=0.3, seed=11, call=2)
    return y + total


def _add_alone(x, r, w, b):
    return add_layer_norm(x, r, w, b)[0]


def _drop(x, r, w, b):
    return dropout(x, 0.3, 5, residual=r) * w + b


def _drop_alone(x, r, w, b):
    return dropout(x, 0.3, 5)


def _policy(x, r, w, b):
    loss, stats = policy_loss(x, r, w.sum().expand(x.shape[:-1]), r > -0.5, x.detach() * 1.1,
                              kl_weight=0.1, return_stats=True)
    return loss + stats[3] * 0


def _policy_each(x, r, w, b):
    return policy_loss(x, r, r, reduction="none")


CALLS = {f.__name__[1:]: (f, names) for f, names in (
    (_norm, ("layer_norm",)), (_norm_mixed, ("layer_norm",)), (_add, ("layer_norm",)),
    (_add_alone, ("layer_norm",)), (_drop, ("dropout",)), (_drop_alone, ("dropout",)),
    (_policy, ("policy_loss",)), (_policy_each, ("policy_loss",)))}


def _inputs(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, r = (torch.randn((4, 25, 72), generator=g, device="cuda") for _ in range(2))
    w, b = (torch.randn(72, generator=g, device="cuda") for _ in range(2))
    return [t.requires_grad_() for t in (x, r, w, b)]


def _grads(out, inputs):
    return torch.autograd.grad(out.float().sum(), inputs, allow_unused=True)


def _same(got, want):
    assert len(got) == len(want)
    for p, q in zip(got, want):
        assert (p is None) == (q is None)
        assert p is None or torch.equal(p, q)


@pytest.mark.parametrize("name", CALLS)
def test_make_fx(name):
    call, ops = CALLS[name]

    def f(*inputs):
        out = call(*inputs)
        return (out, *[g for g in _grads(out, inputs) if g is not None])

    graph = make_fx(f)(*_inputs(0))
    targets = [node.target for node in graph.graph.nodes]
    for op in ops:
        assert getattr(OPS, op).default in targets
        assert getattr(OPS, op + "_backward").default in targets
    for seed in (1, 2):
        inputs = _inputs(seed)
        _same(graph(*inputs), f(*inputs))


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("how", ["make_fx before dispatch", "jit.trace"])
@pytest.mark.parametrize("name", CALLS)
def test_forward_graphs(name, how):
    call, ops = CALLS[name]
    if how == "jit.trace":
        graph = torch.jit.trace(call, tuple(_inputs(0)))
        assert all(f"luma_amd::{op}" in str(graph.graph) for op in ops)
    else:
        graph = make_fx(call, pre_dispatch=True)(*_inputs(0))
        assert all(getattr(OPS, op).default in [n.target for n in graph.graph.nodes] for op in ops)
    for seed in (1, 2):
        inputs = _inputs(seed)
        got, want = graph(*inputs), call(*inputs)
        assert torch.equal(got, want)
        _same(_grads(got, inputs), _grads(want, inputs))


@pytest.mark.parametrize("pre_dispatch", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_make_fx_of_the_backward_alone(name, pre_dispatch):
    """The forward ran before the tracer began."""
    call, ops = CALLS[name]
    inputs = _inputs(3)
    out = call(*inputs)

    def f(g):
        got = torch.autograd.grad(out, inputs, g, retain_graph=True, allow_unused=True)
        return [t for t in got if t is not None]

    graph = make_fx(f, pre_dispatch=pre_dispatch)(torch.ones_like(out))
    targets = [node.target for node in graph.graph.nodes]
    assert all(getattr(OPS, op + "_backward").default in targets for op in ops)
    for seed in (4, 5):
        g = torch.rand(out.shape, generator=torch.Generator(device="cuda").manual_seed(seed),
                       device="cuda").to(out.dtype)
        _same(graph(g), f(g))


def test_dispatch_modes_see_both_directions():
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func)
            return func(*args, **(kwargs or {}))

    for call, ops in CALLS.values():
        inputs = _inputs(6)
        want = call(*inputs)
        want_grads = _grads(want, inputs)
        seen.clear()
        with Mode():
            out = call(*inputs)
            grads = _grads(out, inputs)
        for op in ops:
            assert getattr(OPS, op).default in seen
            assert getattr(OPS, op + "_backward").default in seen
        assert torch.equal(out, want)
        _same(grads, want_grads)


def _model(x, r, w, b):
    y = layer_norm(x, w, b)
    y, x = add_layer_norm(y * 0.5, x, w, b, p=0.2, seed=3, call=1)
    z = dropout(y, 0.2, 3, 2, residual=x)
    return policy_loss(z, r, r, r > -1.0, z.detach() * 0.9, kl_weight=0.1)


@pytest.mark.parametrize("dynamic", [False, True])
def test_compile(dynamic):
    compiled = torch.compile(_model, fullgraph=True, dynamic=dynamic)
    for seed in (0, 1):
        inputs = _inputs(seed)
        want, got = _model(*inputs), compiled(*inputs)
        assert abs(float(got) - float(want)) <= 1e-6 * abs(float(want))
        for p, q in zip(_grads(got, inputs), _grads(want, inputs)):
            assert (p is None) == (q is None)
            # (the compiler fuses and reorders what stands between the operators)
            assert p is None or float((p - q).norm()) <= 1e-5 * float(q.norm())


def test_compile_with_seeds():
    """A seed as a number that changes from call to call, and one on the device."""
    @torch.compile(fullgraph=True)
    def f(x, r, seed):
        return add_layer_norm(dropout(x, 0.3, seed, 1), r, p=0.4, seed=seed, call=2)[0]

    x, r, _, _ = (t.detach() for t in _inputs(9))
    for seed in (3, 4, -5, (1 << 63) - 1):
        want = add_layer_norm(dropout(x, 0.3, seed, 1), r, p=0.4, seed=seed, call=2)[0]
        assert torch.equal(f(x, r, seed), want)
        assert torch.equal(f(x, r, torch.tensor(seed, device="cuda")), want)


@pytest.mark.parametrize("name", CALLS)
def test_functional_transforms_are_refused(name):
    """torch.func does not see through the operators' gradients: it says so."""
    call, _ = CALLS[name]
    plain = [t.detach() for t in _inputs(7)]
    with pytest.raises(RuntimeError, match="functorch|torch.func|vmap"):
        torch.func.grad(lambda *a: call(*a).float().sum())(*plain)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name, grad):
    """A tangent is not lost without a word."""
    call, _ = CALLS[name]
    plain = [t.detach() for t in _inputs(7)]
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = torch.autograd.forward_ad.make_dual(plain[0], torch.ones_like(plain[0]))
        with pytest.raises(RuntimeError, match="jvp|forward AD|forward-mode"):
            call(dual, *plain[1:])


def test_opcheck():
    x, r, w, b = _inputs(8)
    seed = torch.tensor(3, device="cuda")
    check = ("test_schema", "test_faketensor")
    for args in ((x, None, w, b, None, 1e-5, 0.0, 0, 0, 1), (x, r, w, None, seed, 1e-5, 0.2, 0, 1, 0),
                 (x[0, :0], None, None, b, None, 1e-5, 0.0, 0, 0, 2)):
        torch.library.opcheck(OPS.layer_norm.default, args, test_utils=check)
    torch.library.opcheck(OPS.dropout.default, (x, r, seed, 0.2, 0, 1), test_utils=check)
    for reduction in range(4):
        torch.library.opcheck(OPS.policy_loss.default,
                              (x, r, r, r > 0, None, 0.2, 0.2, 0.1, reduction,
                               reduction > 1), test_utils=check)
