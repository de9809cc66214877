"""Global gradient norm and clipping against 64-bit arithmetic.

Tolerances.  The norm is summed in float64 and rounded once to float32: within
one unit of 2^-24 of the exact value (1.01 of it, for the float64 sum's own
rounding).  Clipping: the factor is formed in float32 from the returned norm
by one addition and one division, and each product is rounded once in
float32 and once in the gradient's type; the host does the same operations, so
the gradients are equal bit for bit."""

import math

import numpy as np
import pytest
import torch

import luma_amd
from luma_amd import _lib as L

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NORMS = [2.0, 1.0, math.inf]
SIZES = {
    "one": [1],
    "tiny": [1, 2, 3, 7, 8, 9, 63, 64, 65],
    "tiles": [2047, 2048, 2049, 4096, 511, 512, 513],
    "ragged": [70001, 1, 300007, 5, 12345, 2048 * 33],
    "empty among": [0, 17, 0, 4097],
    "two launches": [100 + i for i in range(L.GRADS_INLINE + 3)],
    "many": [1 + (i * 7919) % 5000 for i in range(3000)],
}


def _exact_norm(grads, p):
    flat = torch.cat([g.detach().double().reshape(-1).cpu() for g in grads])
    return float(torch.linalg.vector_norm(flat, p)) if flat.numel() else 0.0


def _factor(total, max_norm):
    """The clip factor as float32 arithmetic gives it from the norm."""
    with np.errstate(all="ignore"):
        c = np.float32(max_norm) / (np.float32(total) + np.float32(1e-6))
    return np.float32(1.0) if c > 1 else c


def _clipped(g, c):
    return (g.float() * torch.tensor(c, device=g.device)).to(g.dtype)


def _params(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        out.append(p)
    return out


def _near(got, want):
    assert got.dtype == torch.float32 and got.dim() == 0 and got.is_cuda
    assert abs(float(got) - want) <= 1.01 * 2.0 ** -24 * want, (float(got), want)


def _make(sizes, dtype, seed=0, std=0.1):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * std).to(dtype).cuda() for n in sizes]


@pytest.mark.parametrize("p", NORMS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", SIZES)
def test_norm_and_clip(name, dtype, p):
    grads = _make(SIZES[name], dtype)
    want = _exact_norm(grads, p)
    _near(luma_amd.get_total_norm(grads, p), want)
    before = [g.clone() for g in grads]
    total = luma_amd.clip_grad_norm_(_params(grads), 0.37 * want, p)
    _near(total, want)
    c = _factor(float(total), 0.37 * want)
    for g, b in zip(grads, before):
        assert torch.equal(g, _clipped(b, c))


@pytest.mark.parametrize("dtype", DTYPES)
def test_below_the_limit_nothing_is_written(dtype):
    grads = _make([5, 4099], dtype)
    before = [g.clone() for g in grads]
    for limit in (1e9, math.inf):
        luma_amd.clip_grad_norm_(_params(grads), limit)
        assert all(torch.equal(g, b) for g, b in zip(grads, before))


def test_limit_of_zero_clears():
    grads = _make([5, 4099], torch.float32)
    luma_amd.clip_grad_norm_(_params(grads), 0.0)
    assert all(not g.any() for g in grads)


def test_no_gradients():
    p = torch.nn.Parameter(torch.ones(3, device="cuda"))
    assert float(luma_amd.clip_grad_norm_([p], 1.0)) == 0.0
    assert float(luma_amd.get_total_norm([])) == 0.0
    assert float(luma_amd.get_total_norm([torch.empty(0, device="cuda")])) == 0.0
    luma_amd.clip_grads_with_norm_([p], 1.0, torch.tensor(2.0))


@pytest.mark.parametrize("scale", [1e30, 1e-30, 3e-42])
def test_squares_beyond_float32(scale):
    """Squares that overflow or vanish in float32 are summed in float64."""
    x = torch.arange(1, 5001, dtype=torch.float64) * scale / 5000
    g = x.float().cuda()
    want = float(torch.linalg.vector_norm(g.double().cpu()))
    got = float(luma_amd.get_total_norm([g]))
    # (3e-42 lies among float32's subnormal numbers, which are 2^-149 apart)
    assert abs(got - want) <= 1.01 * 2.0 ** -24 * want + 2.0 ** -150


def test_mixed_types_in_one_call():
    grads = [_make([1000 + i], d, seed=i)[0] for i, d in enumerate(DTYPES * 3)]
    want = _exact_norm(grads, 2.0)
    before = [g.clone() for g in grads]
    total = luma_amd.clip_grad_norm_(_params(grads), 1.0)
    _near(total, want)
    c = _factor(float(total), 1.0)
    assert all(torch.equal(g, _clipped(b, c)) for g, b in zip(grads, before))


@pytest.mark.parametrize("p", NORMS)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("at", [0, 2049, 4102])
def test_not_finite(value, at, p):
    g = _make([4103], torch.float32)[0]
    g[at] = value
    grads = [g, _make([300], torch.bfloat16)[0]]
    total = float(luma_amd.get_total_norm(grads, p))
    assert math.isnan(total) if math.isnan(value) else total == math.inf
    with pytest.raises(RuntimeError, match="non-finite"):
        luma_amd.get_total_norm(grads, p, error_if_nonfinite=True)
    before = [x.clone() for x in grads]
    with pytest.raises(RuntimeError, match="non-finite"):
        luma_amd.clip_grad_norm_(_params(grads), 1.0, p, error_if_nonfinite=True)
    assert all(torch.equal(x.view(torch.int16), b.view(torch.int16))
               for x, b in zip(grads, before))
    luma_amd.clip_grad_norm_(_params(grads), 1.0, p)
    c = _factor(total, 1.0)        # 0 for an infinite norm, NaN for NaN
    for x, b in zip(grads, before):
        torch.testing.assert_close(x, _clipped(b, c), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [1, 3, 5, 7])
def test_views_off_every_boundary(dtype, offset):
    """Gradients packed without padding; what lies around them stays."""
    sizes = [offset, 1001, 4096, 3, 9999]
    flat = _make([sum(sizes) + 16], dtype)[0]
    before, views, at = flat.clone(), [], 1
    for n in sizes:
        views.append(flat[at:at + n])
        at += n
    total = luma_amd.clip_grad_norm_(_params(views), 0.5)
    _near(total, _exact_norm([before[1:at]], 2.0))
    c = _factor(float(total), 0.5)
    assert torch.equal(flat[1:at], _clipped(before[1:at], c))
    assert flat[0] == before[0] and torch.equal(flat[at:], before[at:])


def test_layouts():
    """Dense tensors of any element order in place; others by a copy."""
    base = _make([6 * 5 * 4 * 8], torch.float32)[0]
    last = base.clone().view(6, 5, 4, 8).to(memory_format=torch.channels_last)
    turned = base.clone().view(30, 32).t()
    sliced = base.clone().view(30, 32)[:, 3:17]
    for g in (last, turned, sliced):
        before, want = g.clone(), _exact_norm([g], 2.0)
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        _near(luma_amd.get_total_norm([g]), want)
        total = luma_amd.clip_grad_norm_([p], 0.5 * want)
        assert torch.equal(g, _clipped(before, _factor(float(total), 0.5 * want)))


def test_expanded_gradient():
    """A broadcast gradient counts every element; it has no place to be clipped in."""
    g = torch.full((1,), 2.0, device="cuda").expand(1000)
    _near(luma_amd.get_total_norm([g]), math.sqrt(4000.0))


def test_listed_twice_counts_once():
    g = _make([5000], torch.float32)[0]
    before, want = g.clone(), _exact_norm([g], 2.0)
    p = _params([g])[0]
    total = luma_amd.clip_grad_norm_([p, p], 0.5 * want)
    _near(total, want)
    assert torch.equal(g, _clipped(before, _factor(float(total), 0.5 * want)))
    _near(luma_amd.get_total_norm([g, g]), math.sqrt(2.0) * _exact_norm([g], 2.0))


def test_shared_memory_is_refused():
    flat = _make([1000], torch.float32)[0]
    before = flat.clone()
    with pytest.raises(ValueError, match="share memory"):
        luma_amd.clip_grad_norm_(_params([flat[:600], flat[500:], flat[:10]]), 0.1)
    assert torch.equal(flat, before)


def test_refusals():
    p = _params(_make([10], torch.float32))
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            luma_amd.clip_grad_norm_(p, bad)
    for bad in (3.0, 0.0, -math.inf):
        with pytest.raises(ValueError, match="norm_type"):
            luma_amd.clip_grad_norm_(p, 1.0, bad)
        with pytest.raises(ValueError, match="norm_type"):
            luma_amd.get_total_norm([p[0].grad], bad)
    with pytest.raises(ValueError, match="dtype"):
        luma_amd.get_total_norm([torch.ones(3, device="cuda", dtype=torch.float64)])
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        luma_amd.get_total_norm([torch.ones(3)])
    with pytest.raises(RuntimeError, match="sparse"):
        luma_amd.get_total_norm([torch.ones(3, device="cuda").to_sparse()])
    with pytest.raises(ValueError, match="one-element"):
        luma_amd.clip_grads_with_norm_(p, 1.0, torch.ones(2, device="cuda"))


def test_scale_by_a_known_norm():
    grads = _make([100, 5000, 3], torch.bfloat16)
    before = [g.clone() for g in grads]
    total = luma_amd.get_total_norm(grads)
    luma_amd.clip_grads_with_norm_(_params(grads), 0.2, total)
    c = _factor(float(total), 0.2)
    assert all(torch.equal(g, _clipped(b, c)) for g, b in zip(grads, before))


def test_parameters_without_gradient_and_a_generator():
    grads = _make([100, 200], torch.float32)
    params = _params(grads)
    params.insert(1, torch.nn.Parameter(torch.ones(5, device="cuda")))
    want = _exact_norm(grads, 2.0)
    _near(luma_amd.clip_grad_norm_((q for q in params), 1e9), want)
    _near(luma_amd.clip_grad_norm_(params[0], 1e9), _exact_norm(grads[:1], 2.0))


def test_same_bits_every_time():
    grads = _make([100003] * 20 + [7] * 300, torch.float32)
    totals = {float(luma_amd.get_total_norm(grads)) for _ in range(10)}
    assert len(totals) == 1


def test_without_the_host_module(monkeypatch):
    """The path over any tensors gives what the quick one gives."""
    a, b = (_make(SIZES["ragged"], torch.bfloat16) for _ in range(2))
    t = luma_amd.clip_grad_norm_(_params(a), 1.0)
    monkeypatch.setattr(luma_amd.clip, "_host", lambda: None)
    u = luma_amd.clip_grad_norm_(_params(b), 1.0)
    assert torch.equal(t, u) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("tensors", [3, 700])
def test_autograd_sees_the_write(tensors):
    grads = _make([17] * tensors + [5], torch.float32)
    before = [g._version for g in grads]
    luma_amd.get_total_norm(grads)
    assert [g._version for g in grads] == before
    luma_amd.clip_grad_norm_(_params(grads), 0.1)
    assert all(g._version > v for g, v in zip(grads, before))


def test_other_stream():
    grads = _make([1 << 20] * 4, torch.float32)
    want = _exact_norm(grads, 2.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for g in grads:
            g.mul_(2.0)
        total = luma_amd.clip_grad_norm_(_params(grads), 1.0)
    s.synchronize()
    _near(total, 2.0 * want)
    assert abs(_exact_norm(grads, 2.0) - 1.0) < 1e-5


@pytest.mark.parametrize("tensors", [3, L.GRADS_INLINE + 5])
def test_graph(tensors):
    """A captured call clips whatever the gradients hold at each replay."""
    grads = _make([997] * tensors, torch.float32)
    params = _params(grads)
    luma_amd.clip_grad_norm_(params, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total = luma_amd.clip_grad_norm_(params, 1.0)
    for seed in range(1, 5):
        new = _make([997] * tensors, torch.float32, seed=seed)
        for g, x in zip(grads, new):
            g.copy_(x)
        want = [x.clone() for x in new]
        t = luma_amd.clip_grad_norm_(_params(want), 1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(total) - float(t)) <= 2.0 ** -23 * float(t)
        c = _factor(float(total), 1.0)
        assert all(torch.equal(g, _clipped(x, c)) for g, x in zip(grads, new))


def test_elements_past_32_bits():
    n = 2 ** 31 + 2053
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[0], g[2 ** 31 + 5], g[n - 1] = 3.0, 4.0, 12.0
    _near(luma_amd.get_total_norm([g]), 13.0)
    luma_amd.clip_grad_norm_(_params([g]), 6.5)
    assert [float(g[i]) for i in (0, 2 ** 31 + 5, n - 1)] == [1.5, 2.0, 6.0]


def test_sharded_gradients():
    """DTensors over a mesh of one rank: the local shards' sums joined."""
    import socket

    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import Partial, Replicate, Shard, distribute_tensor, DTensor

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cuda", (1,))
        grads = _make([6400, 330, 17], torch.float32)
        want = _exact_norm(grads, 2.0)
        places = [[Shard(0)], [Replicate()], None]
        params = []
        for g, place in zip(grads, places):
            g = g if place is None else distribute_tensor(g, mesh, place)
            p = torch.nn.Parameter(torch.empty_like(g))
            p.grad = g
            params.append(p)
        before = [p.grad._local_tensor.clone() if hasattr(p.grad, "_local_tensor")
                  else p.grad.clone() for p in params]
        total = luma_amd.clip_grad_norm_(params, 0.5 * want)
        _near(total, want)
        c = _factor(float(total), 0.5 * want)
        for p, b in zip(params, before):
            local = getattr(p.grad, "_local_tensor", p.grad)
            assert torch.equal(local, _clipped(b, c))
        _near(luma_amd.get_total_norm([p.grad for p in params], math.inf),
              _exact_norm([p.grad.full_tensor() if hasattr(p.grad, "full_tensor") else p.grad
                           for p in params], math.inf))
        half = DTensor.from_local(grads[0], mesh, [Partial()])
        with pytest.raises(ValueError, match="Partial"):
            luma_amd.get_total_norm([half])
    finally:
        dist.destroy_process_group()
