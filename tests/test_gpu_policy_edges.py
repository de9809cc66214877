"""policy_loss where a token's terms leave float32's range: probabilities of 0,
ratios past exp(88.7), advantages of 0, a KL term that is only a figure."""

import itertools
import math

import pytest
import torch

from luma_amd import _lib as L
from luma_amd import policy_loss

pytestmark = pytest.mark.gpu

REDUCTIONS = ["mean", "sequence", "sum", "none"]
LENGTHS = [1, 3, 50, 1500]      # one launch, tokens one by one, pieces of rows
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _tokens(length, dtype, at, **places):
    """Three rows of ordinary tokens; `places`: what stands at token `at` of row 1."""
    g = torch.Generator(device="cuda").manual_seed(length)
    shape = (3, length)
    t = {"logp": torch.rand(shape, generator=g, device="cuda").add_(1e-3).log_()}
    t["old"] = t["logp"] + torch.randn(shape, generator=g, device="cuda") * 0.1
    t["ref"] = t["logp"] + torch.randn(shape, generator=g, device="cuda") * 0.1
    t = {name: v.to(dtype) for name, v in t.items()}
    t["advantage"] = torch.randn(shape, generator=g, device="cuda")
    for name, value in places.items():
        t[name][1, at] = value
    t["logp"].requires_grad_()
    return t


def _loss(t, ref=True, **kw):
    return policy_loss(t["logp"], t["old"], t["advantage"], None, t["ref"] if ref else None, **kw)


def _with_grad(t, loss):
    g = torch.Generator(device="cuda").manual_seed(1)
    out = torch.rand(loss.shape, generator=g, device="cuda") + 0.5
    return loss.detach(), torch.autograd.grad(loss, t["logp"], out)[0]


@pytest.fixture(params=["the host module", "operators"])
def path(request, monkeypatch):
    if request.param == "operators":
        monkeypatch.setattr(L, "host_calls", lambda: None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", LENGTHS)
@pytest.mark.parametrize("logp,ref", [(-math.inf, -1.0), (-200.0, -1.0), (-1.0, math.inf),
                                      (-1.0, math.nan)])
def test_a_weight_of_0_leaves_the_term_out(path, logp, ref, length, dtype):
    """Loss and gradient are those without a reference, bit for bit, whatever exp(q) is."""
    t = _tokens(length, dtype, length // 2, logp=logp, ref=ref)
    for reduction in REDUCTIONS:
        want = _with_grad(t, _loss(t, False, reduction=reduction))
        assert all(bool(v.isfinite().all()) for v in want)
        for figures in (False, True):
            loss = _loss(t, reduction=reduction, kl_weight=0.0, return_stats=figures)
            if figures:
                loss, stats = loss
                # (the figure is the divergence's all the same)
                assert not bool(stats[1].isfinite())
            assert all(torch.equal(p, q) for p, q in zip(_with_grad(t, loss), want)), reduction


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", LENGTHS)
@pytest.mark.parametrize("old", [-200.0, -math.inf])
def test_an_advantage_of_0(path, old, length, dtype):
    """min(r A, clip(r) A) is 0, and so is its gradient, past float32's largest ratio too;
    the other tokens are as beside an ordinary ratio."""
    at = length // 2
    for reduction, high in itertools.product(REDUCTIONS, (0.2, math.inf)):
        got, want = [], []
        for values, token in ((got, old), (want, -1.0)):
            t = _tokens(length, dtype, at, logp=-1.0, old=token, advantage=0.0)
            values += _with_grad(t, _loss(t, False, clip_high=high, reduction=reduction))
        assert bool(want[0].isfinite().all()) and bool(want[1].isfinite().all())
        assert all(torch.equal(p, q) for p, q in zip(got, want)), (reduction, high)
        assert float(got[1][1, at]) == 0.0
        if reduction == "none":
            assert float(got[0][1, at]) == 0.0
        # (an advantage for each row, and what is no number stays none)
        t = _tokens(length, dtype, at, logp=-1.0, old=old)
        zero = torch.tensor([1.0, 0.0, 1.0], device="cuda")
        loss = policy_loss(t["logp"], t["old"], zero, clip_high=high, reduction=reduction)
        assert bool(loss.isfinite().all())
        t = _tokens(length, dtype, at, logp=math.nan, old=old, advantage=0.0)
        assert bool(_loss(t, False, clip_high=high, reduction=reduction).sum().isnan())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", LENGTHS)
def test_infinite_divergences(path, length, dtype):
    """exp(x) - 1 - x grows without end: an infinite x has an infinite one."""
    at = length // 2
    t = _tokens(length, dtype, at, logp=-1.0, old=-math.inf, advantage=2.0)
    loss, stats = _loss(t, False, clip_high=0.25, reduction="none", return_stats=True)
    assert float(loss[1, at].detach()) == -2.5 and float(stats[2]) == math.inf
    for low in (-math.inf, -200.0):
        t = _tokens(length, dtype, at, logp=low, ref=-1.0)
        loss, stats = _loss(t, kl_weight=0.5, reduction="none", return_stats=True)
        assert float(loss[1, at].detach()) == math.inf and float(stats[1]) == math.inf
        d, = torch.autograd.grad(loss.sum(), t["logp"])
        assert float(d[1, at]) == -math.inf
        loss = _loss(t, kl_weight=0.5)
        assert float(loss.detach()) == math.inf
    # (a probability of 0 that was one before: a ratio of 0, which has moved as far)
    t = _tokens(length, dtype, at, logp=-math.inf, old=-1.0)
    assert float(_loss(t, False, return_stats=True)[1][2]) == math.inf
