"""Captured norms and clippings of lists long enough for a device table, which
go without one under capture: nothing is allocated on the host, and every
replay gives what the eager call gives.  (The eager call sums in another order,
so norms are within one unit of 2^-23; the gradients follow from the norm bit
for bit, as in the eager call's tests.)"""

import numpy as np
import pytest
import torch

import luma_amd
from luma_amd import LUMA

pytestmark = pytest.mark.gpu

SIZES = [1 + (i * 37) % 3000 for i in range(700)]
NO_TABLE = luma_amd.clip.NO_TABLE


def _grads(seed, std=0.1):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * std).cuda() for n in SIZES]


def _params(grads):
    out = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(out, grads):
        p.grad = g
    return out


@pytest.fixture
def pinned(monkeypatch):
    """Pinned allocations, counted."""
    count, empty, pin = [0], torch.empty, torch.Tensor.pin_memory

    def counted(*args, **more):
        count[0] += bool(more.get("pin_memory"))
        return empty(*args, **more)

    def counted_pin(*args, **more):
        count[0] += 1
        return pin(*args, **more)

    monkeypatch.setattr(torch, "empty", counted)
    monkeypatch.setattr(torch.Tensor, "pin_memory", counted_pin)
    return count


@pytest.mark.parametrize("module", [True, False])
@pytest.mark.parametrize("call", ["get_total_norm", "clip_grad_norm_", "clip_grads_with_norm_"])
def test_captured_call(call, module, pinned, monkeypatch):
    assert len(SIZES) > NO_TABLE
    if not module:
        monkeypatch.setattr(luma_amd.clip, "_host", lambda: None)
    grads = _grads(0)
    params = _params(grads)
    known = torch.tensor(2.5, device="cuda")

    def run(params, grads):
        if call == "get_total_norm":
            return luma_amd.get_total_norm(grads)
        if call == "clip_grad_norm_":
            return luma_amd.clip_grad_norm_(params, 1.0)
        luma_amd.clip_grads_with_norm_(params, 1.0, known)
        return known

    run(params, grads)
    eager = pinned[0]
    assert eager > 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total = run(params, grads)
    assert pinned[0] == eager
    for seed in range(1, 5):
        new = _grads(seed)
        for g, x in zip(grads, new):
            g.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        copies = [x.clone() for x in new]
        want = run(_params(copies), copies)
        assert abs(float(total) - float(want)) <= 2.0 ** -23 * float(want)
        if call == "get_total_norm":
            assert all(torch.equal(g, x) for g, x in zip(grads, new))
            continue
        c = np.float32(1.0) / (np.float32(float(total)) + np.float32(1e-6))
        c = torch.tensor(min(c, np.float32(1.0)), device="cuda")
        assert all(torch.equal(g, x * c) for g, x in zip(grads, new))


def test_captured_step_with_other_gradients_than_the_last_eager_one():
    """Two gradient buffers in turn; the step that reads the first is captured
    after an eager one that read the second: its rows go as launch arguments."""
    a, b = _params(_grads(0)), _params(_grads(0))
    one, two = _grads(1), _grads(2)
    opts = []
    for params in (a, b):
        opt = LUMA(params, lr=1e-3, max_grad_norm=0.5)
        opt._base_seed = 0x1234567
        opts.append(opt)

    def step(opt, params, grads):
        for p, g in zip(params, grads):
            p.grad = g
        opt.step()

    for opt, params in zip(opts, (a, b)):
        for grads in (one, two, one, two):
            step(opt, params, grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(opts[0], a, one)
    for t in range(4):
        for g, x in zip(one, _grads(10 + t, 0.05 * (t + 1))):
            g.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got = float(opts[0].grad_norm)
        want = float(sum((g.double() ** 2).sum() for g in one)) ** 0.5
        assert abs(got - want) <= 1.01 * 2.0 ** -24 * want
        # a step that the same scale clips
        opts[1].max_grad_norm = None
        norm = opts[0].grad_norm.cpu()
        c = torch.tensor(0.5) / (norm + torch.tensor(1e-6))
        opts[1].grad_scale = (torch.tensor(1.0) / c.clamp(max=1.0)).cuda()
        step(opts[1], b, one)
        torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
