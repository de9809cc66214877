"""LUMA(max_grad_norm=...) where this rank's shard of a DTensor is empty (a mesh
of one rank; the reductions are counted): each step joins the norm's
reductions, and steps what it has as plain parameters are stepped."""

import socket

import pytest
import torch
import torch.distributed as dist

import luma_amd
from luma_amd import LUMA

pytestmark = pytest.mark.gpu


@pytest.fixture
def mesh():
    from torch.distributed.device_mesh import init_device_mesh

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1)
    try:
        yield init_device_mesh("cuda", (1,))
    finally:
        dist.destroy_process_group()


@pytest.fixture
def joined(monkeypatch):
    """The norms' reductions, counted."""
    calls, join = [], luma_amd.clip._join_shards

    def counted(power, code, mesh, dims):
        calls.append(dims)
        join(power, code, mesh, dims)

    monkeypatch.setattr(luma_amd.clip, "_join_shards", counted)
    return calls


def _empty(mesh):
    from torch.distributed.tensor import DTensor, Shard

    def shard():
        return DTensor.from_local(torch.empty((0, 6), device="cuda"), mesh, [Shard(0)])

    p = torch.nn.Parameter(shard())
    p.grad = shard()
    return p


def _plain(seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.nn.Parameter((torch.randn((40, 30), generator=g) * 0.02).cuda())
    p.grad = torch.randn((40, 30), generator=g).cuda()
    return p


def _opt(params, **more):
    opt = LUMA(params, lr=1e-3, **more)
    opt._base_seed = 0x1234567
    return opt


def test_empty_shard_beside_a_plain_parameter(mesh, joined):
    p, q = _plain(0), _plain(0)
    # (the parameters' numbers key the rounding's draws: the plain one comes first)
    a, b = _opt([p, _empty(mesh)], max_grad_norm=1.0), _opt([q], max_grad_norm=1.0)
    for t in range(1, 5):
        a.step()
        b.step()
        assert joined == [(0,)] * t
        assert torch.equal(a.grad_norm, b.grad_norm)
    assert torch.equal(p, q)


def test_only_an_empty_shard(mesh, joined):
    opt = _opt([_empty(mesh)], max_grad_norm=1.0)
    for t in range(1, 3):
        opt.step()
        assert joined == [(0,)] * t
        assert float(opt.grad_norm) == 0.0
    opt.grad_scale = torch.tensor(8.0, device="cuda")
    opt.step()
    assert float(opt.grad_norm) == 0.0
    opt.max_grad_norm = None
    opt.step()
    assert len(joined) == 3


def test_gradients_that_the_step_promotes(mesh, joined):
    """float64 gradients count as the float32 ones that the step takes them as."""
    from torch.distributed.tensor import Shard, distribute_tensor

    q = _plain(0)
    p = torch.nn.Parameter(distribute_tensor(q.detach().clone(), mesh, [Shard(0)]))
    p.grad_dtype = q.grad_dtype = None
    g = q.grad.double()
    p.grad, q.grad = distribute_tensor(g, mesh, [Shard(0)]), g
    a, b = _opt([p], max_grad_norm=1.0), _opt([q], max_grad_norm=1.0)
    for t in range(1, 3):
        a.step()
        b.step()
        assert joined == [(0,)] * t and torch.equal(a.grad_norm, b.grad_norm)
    assert torch.equal(p.detach().to_local(), q.detach())


def test_sharded_factor_is_the_plain_one(mesh, joined):
    """The factor of a joined norm is the same division as the kernel's, so that a
    sharded parameter's step is the plain one's, bit for bit."""
    from torch.distributed.tensor import Shard, distribute_tensor

    q = _plain(0)
    p = torch.nn.Parameter(distribute_tensor(q.detach().clone(), mesh, [Shard(0)]))
    a, b = _opt([p]), _opt([q])
    g = q.grad
    for t in range(24):
        q.grad = g * (1.0 + 0.37 * t)
        p.grad = distribute_tensor(q.grad, mesh, [Shard(0)])
        for opt in (a, b):
            opt.max_grad_norm = 0.3 + 0.11 * t
            opt.grad_scale = torch.tensor(3.0 + t, device="cuda")
            opt.step()
        assert torch.equal(a.grad_norm, b.grad_norm)
        assert torch.equal(p.detach().to_local(), q.detach()), t
