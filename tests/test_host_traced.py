"""Calls that a tracer or a dispatch mode watches, without a GPU: they go to the
operators, which it sees, and not to the host module, whose kernels it does
not (a recorded graph would hold the allocation of their outputs alone)."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

import luma_amd
from luma_amd import _lib as L
from luma_amd import linear_cross_entropy


class Seen(TorchDispatchMode):
    """A dispatch mode that changes nothing, as an operator counter is one."""

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def _in_mode(f, x):
    with Seen():
        f(x)


WAYS = {"make_fx": lambda f, x: make_fx(f)(x),
        "make_fx before dispatch": lambda f, x: make_fx(f, pre_dispatch=True)(x),
        "jit.trace": lambda f, x: torch.jit.trace(f, x, check_trace=False),
        "dispatch mode": _in_mode}


@pytest.mark.parametrize("how", WAYS)
def test_loss_goes_to_the_operator(how, monkeypatch):
    """(On the CPU the check of the device, behind the choice, is what answers.)"""
    calls = []

    class Host:
        @staticmethod
        def xent(hidden, weight, target, ignore_index, reduction):
            calls.append(1)
            return hidden.sum()

    monkeypatch.setattr(L, "host_calls", lambda: Host)
    w, t = torch.ones(6, 8), torch.zeros(4, dtype=torch.int64)

    def f(x):
        return linear_cross_entropy(x, w, t)

    f(torch.ones(4, 8))
    assert calls == [1]                 # eager: the host module
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        WAYS[how](f, torch.ones(4, 8))
    assert calls == [1]


def _clip(x):
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = x
    return luma_amd.clip_grad_norm_([p], 1.0)


def _scale(x):
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = x
    luma_amd.clip_grads_with_norm_([p], 1.0, torch.tensor(2.0))
    return x


@pytest.mark.parametrize("how", ["make_fx", "make_fx before dispatch", "jit.trace"])
@pytest.mark.parametrize("f", [lambda x: luma_amd.get_total_norm([x]), _clip, _scale],
                         ids=["get_total_norm", "clip_grad_norm_", "clip_grads_with_norm_"])
def test_norm_and_clipping_refuse_a_tracer(f, how):
    """They are no operators: a graph of them would return memory that nothing fills."""
    with pytest.raises(RuntimeError, match="cannot be recorded"):
        WAYS[how](f, torch.ones(3))
