"""Operators called with operands that do not fit each other, as a recorded graph calls
them when it is given others than those that it was recorded with: each call says so
before anything is launched."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from luma_amd import add_layer_norm, dropout, layer_norm, policy_loss
from operands_util import BAD, BF16, CALLS, operands
from operands_util import tensor as _t

pytestmark = pytest.mark.gpu

OPS = torch.ops.luma_amd


@pytest.mark.parametrize("name", CALLS)
def test_what_fits(name):
    out = getattr(OPS, name)(*operands(name))
    torch.cuda.synchronize()
    for t in out if isinstance(out, (tuple, list)) else [out]:
        assert bool(t.isfinite().all())


@pytest.mark.parametrize("name,change", [(n, c) for n, cs in BAD.items() for c in cs])
def test_what_does_not_fit(name, change):
    # (a RuntimeError: the library's own refusal)
    with pytest.raises((ValueError, RuntimeError)):
        getattr(OPS, name)(*operands(name, change))


@pytest.mark.parametrize("name,key", [(n, k) for n, ops in CALLS.items() for k, v in ops.items()
                                      if callable(v)] + [("dropout", "seed"), ("layer_norm", "seed")])
def test_another_device(name, key):
    args = operands(name)
    at = list(CALLS[name]).index(key)
    args[at] = torch.zeros(1, dtype=torch.int64) if key == "seed" else args[at].cpu()
    with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
        getattr(OPS, name)(*args)


RECORDED = {
    "layer_norm": (lambda x, r, w: layer_norm(x, w),
                   [((6, 20), (6, 20), (24,)), ((6, 48), (6, 48), (24,))]),
    "add_layer_norm": (lambda x, r, w: add_layer_norm(x, r, w, p=0.5, seed=1)[0],
                       [((6, 24), (5, 24), (24,)), ((7, 24), (6, 24), (24,)),
                        ((6, 48), (6, 48), (24,))]),
    "dropout": (lambda x, r, w: dropout(x, 0.5, 1, residual=r), [((9, 24), (6, 24), (24,))]),
    "policy_loss": (lambda x, r, w: policy_loss(x, r, x[:, 0].detach(), r > 0),
                    [((9, 24), (6, 24), (24,)), ((6, 30), (6, 24), (24,))]),
}


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.filterwarnings("ignore::DeprecationWarning")
@pytest.mark.parametrize("how", ["make_fx", "jit.trace"])
@pytest.mark.parametrize("name", RECORDED)
def test_recorded_graphs(name, how):
    call, bad = RECORDED[name]
    inputs = [_t(6, 24), _t(6, 24), _t(24)]
    graph = make_fx(call)(*inputs) if how == "make_fx" else torch.jit.trace(call, tuple(inputs))
    assert torch.equal(graph(*inputs), call(*inputs))
    for shapes in bad:
        with pytest.raises((ValueError, RuntimeError), match="match|advantage"):
            graph(*(_t(*s) for s in shapes))
    other = [_t(6, 24, dtype=BF16), _t(6, 24), _t(24)]
    if name in ("layer_norm", "add_layer_norm", "policy_loss"):
        with pytest.raises((ValueError, RuntimeError)):
            graph(*other)
    assert torch.equal(graph(*inputs), call(*inputs))
