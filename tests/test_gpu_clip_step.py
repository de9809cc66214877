"""LUMA(max_grad_norm=...): clipping inside the step.

A step multiplies each gradient by f32(1 / (double)s), s = scale / factor,
rounded to the gradient's type: exactly what it does with a GradScaler whose
scale is s, so the codes and parameters equal those of such a step bit for
bit.  A factor of 1 leaves the step as it is without clipping, bit for bit."""

import math

import pytest
import torch

import luma_amd
from luma_amd import LUMA

pytestmark = pytest.mark.gpu

HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
SHAPES = [(96, 100), (4097,), (64, 33), (1,), (300, 7)]
MANY = [(1 + (i * 37) % 300,) for i in range(700)]      # a device table of rows


def _params(shapes, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = [(torch.randn(s, generator=g) * 0.02).cuda().requires_grad_(True) for s in shapes]
    for p in out:
        p.grad_dtype = None
    return out


def _grads(shapes, t, dtype, std=0.1):
    g = torch.Generator().manual_seed(100 + t)
    return [(torch.randn(s, generator=g) * std).to(dtype).cuda() for s in shapes]


def _opt(params, **more):
    opt = LUMA(params, **HYPER, **more)
    opt._base_seed = 0x1234567
    return opt


def _norm(grads):
    return math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))


def _equal(a, b, pa, pb):
    sa, sb = a.state_dict()["state"], b.state_dict()["state"]
    for i, (p, q) in enumerate(zip(pa, pb)):
        assert torch.equal(p, q)
        for k in ("Q_m", "Q_w", "S_m", "S_v", "step"):
            x, y = sa[i][k], sb[i][k]
            assert torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y


def _set(params, grads):
    for p, g in zip(params, grads):
        p.grad = g


def _scale(opt, grads, max_norm, scale=1.0):
    """s as the library forms it, in float32 from the norm that it reports."""
    f = torch.float32
    norm = opt.grad_norm.cpu()
    want = _norm(grads) / scale
    assert abs(float(norm) - want) <= 2.02 * 2.0 ** -24 * want
    c = torch.tensor(max_norm, dtype=f) / (norm + torch.tensor(1e-6, dtype=f))
    return (torch.tensor(scale, dtype=f) / c.clamp(max=1.0)).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shapes", [SHAPES, MANY], ids=["few", "many"])
def test_clipped_step(shapes, dtype):
    pa, pb = _params(shapes), _params(shapes)
    a, b = _opt(pa, max_grad_norm=1.0), _opt(pb)
    for t in range(4):
        grads = _grads(shapes, t, dtype)
        before = [g.clone() for g in grads]
        _set(pa, grads)
        _set(pb, grads)
        a.step()
        b.grad_scale = _scale(a, grads, 1.0)
        assert float(b.grad_scale) > 1.5
        b.step()
        assert all(torch.equal(g, x) for g, x in zip(grads, before))
    _equal(a, b, pa, pb)


def test_below_the_limit_it_is_the_plain_step():
    pa, pb = _params(SHAPES), _params(SHAPES)
    a, b = _opt(pa, max_grad_norm=1e6), _opt(pb)
    for t in range(4):
        grads = _grads(SHAPES, t, torch.bfloat16)
        _set(pa, grads)
        _set(pb, grads)
        a.step()
        b.step()
        assert float(a.grad_norm) > 0.0
    _equal(a, b, pa, pb)
    assert b.grad_norm is None


def test_like_clip_grad_norm_():
    """The clipped gradients of both are within three roundings of 2^-24: after
    one step of Adam's size lr the parameters are within lr of a few parts in
    2^-20 (a code that falls on the other side adds at most a grid step,
    2^-15 of the update)."""
    pa, pb = _params(SHAPES), _params(SHAPES)
    a, b = _opt(pa, max_grad_norm=0.5), _opt(pb)
    for t in range(3):
        grads = _grads(SHAPES, t, torch.float32)
        _set(pa, grads)
        _set(pb, [g.clone() for g in grads])
        a.step()
        total = luma_amd.clip_grad_norm_(pb, 0.5)
        b.step()
        assert torch.equal(total, a.grad_norm)
    for p, q in zip(pa, pb):
        assert float((p - q).abs().max()) <= 3 * HYPER["lr"] * 2.0 ** -9


def test_with_grad_scaler():
    pa, pb = _params(SHAPES), _params(SHAPES)
    a, b = _opt(pa, max_grad_norm=0.25), _opt(pb)
    a.grad_scale = torch.tensor(1024.0, device="cuda")
    a.found_inf = torch.tensor(0.0, device="cuda")
    for t in range(3):
        grads = [g * 1024.0 for g in _grads(SHAPES, t, torch.float32)]
        _set(pa, grads)
        _set(pb, grads)
        a.step()
        b.grad_scale = _scale(a, grads, 0.25, 1024.0)
        b.step()
    _equal(a, b, pa, pb)
    before = [p.clone() for p in pa]
    a.found_inf.fill_(1.0)          # an overflowed step does nothing
    pa[0].grad[0, 0] = math.inf
    a.step()
    assert all(torch.equal(p, q) for p, q in zip(pa, before))


def test_set_and_unset():
    params = _params(SHAPES)
    opt = _opt(params)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            opt.max_grad_norm = bad
        with pytest.raises(ValueError, match="max_norm"):
            _opt(params, max_grad_norm=bad)
    assert opt.max_grad_norm is None
    _set(params, _grads(SHAPES, 0, torch.float32))
    opt.step()
    assert opt.grad_norm is None
    opt.max_grad_norm = 1
    opt.step()
    assert abs(float(opt.grad_norm) - _norm([p.grad for p in params])) < 1e-3
    assert "max_grad_norm" not in opt.state_dict()
    assert all("max_grad_norm" not in g for g in opt.param_groups)


@pytest.mark.parametrize("shapes", [SHAPES, MANY], ids=["few", "many"])
def test_graph(shapes):
    """Each replay clips by the norm of the gradients it finds."""
    pa, pb = _params(shapes), _params(shapes)
    a, b = _opt(pa, max_grad_norm=1.0), _opt(pb)
    grads = _grads(shapes, 0, torch.float32)
    _set(pa, grads)
    _set(pb, grads)
    a.step()
    b.grad_scale = _scale(a, grads, 1.0)
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for t in range(1, 5):
        for g, x in zip(grads, _grads(shapes, t, torch.float32, std=0.05 * t)):
            g.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        b.grad_scale = _scale(a, grads, 1.0)
        b.step()
        torch.cuda.synchronize()
    _equal(a, b, pa, pb)


def test_alternating_gradients():
    """A planned step whose gradients move between buffers."""
    pa, pb = _params(MANY), _params(MANY)
    a, b = _opt(pa, max_grad_norm=1.0), _opt(pb)
    sets = [_grads(MANY, k, torch.float32) for k in range(2)]
    for t in range(6):
        _set(pa, sets[t % 2])
        _set(pb, sets[t % 2])
        a.step()
        b.grad_scale = _scale(a, sets[t % 2], 1.0)
        b.step()
    _equal(a, b, pa, pb)


def test_not_finite():
    """As clip_grad_norm_: an infinite norm clears the finite gradients, NaN spreads."""
    params = _params([(100,), (50,)])
    opt = _opt(params, max_grad_norm=1.0)
    grads = _grads([(100,), (50,)], 0, torch.float32)
    grads[0][3] = math.inf
    _set(params, grads)
    opt.step()
    assert float(opt.grad_norm) == math.inf
    assert bool(params[1].isfinite().all())


def test_sharded_parameter():
    """A DTensor over a mesh of one rank: the joined norm, the same step."""
    import socket

    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import Shard, distribute_tensor

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cuda", (1,))
        plain, = _params([(96, 100)])
        spread = torch.nn.Parameter(distribute_tensor(plain.detach().clone(), mesh, [Shard(0)]))
        a, b = _opt([spread], max_grad_norm=1.0), _opt([plain], max_grad_norm=1.0)
        for t in range(3):
            g, = _grads([(96, 100)], t, torch.float32)
            plain.grad = g
            spread.grad = distribute_tensor(g, mesh, [Shard(0)])
            a.step()
            b.step()
            assert torch.equal(a.grad_norm, b.grad_norm)
        assert torch.equal(spread.detach().to_local(), plain.detach())
    finally:
        dist.destroy_process_group()
