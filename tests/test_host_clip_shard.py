"""LUMA(max_grad_norm=...) over shards, two CPU ranks over gloo: in step() every
rank joins the same reductions in the same order, whatever it holds of the
parameters.  Of a parameter of one row rank 0 has the row and rank 1 nothing.
(There is no GPU: a call's power is taken with torch, and a rank that has
something to step is refused behind its norm.)"""

import datetime

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from luma_amd import LUMA, clip, optimizer
from luma_amd import _lib as L

# (shape, mesh): "a" of one dimension, "b" of two, the second sharded; None: a plain tensor
SETS = {"only empty shards": [((1, 6), "a"), ((1, 3), "a")],
        "an empty shard beside a plain parameter": [((0,), None), ((1, 6), "a"), ((5,), None)],
        "an order that the empty shards decide": [((1, 6), "b"), ((8, 3), "a"), ((6, 2), "b")]}


class _Batch(clip._Batch):
    def args(self, norm, max_norm, total, power=None):
        return norm, power

    def call(self, name, args):
        norm, power = args
        assert name == "luma_grad_norm" and norm == L.NORM_L2
        for g in self.hold:
            power += (g.double() ** 2).sum()


def _grads(name, world):
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import Replicate, Shard, distribute_tensor
    meshes = {"a": (init_device_mesh("cpu", (world,)), [Shard(0)]),
              "b": (init_device_mesh("cpu", (1, world)), [Replicate(), Shard(0)])}
    out = []
    for i, (shape, where) in enumerate(SETS[name]):
        g = torch.arange(1.0, 1.0 + torch.Size(shape).numel()).view(shape) * (i + 1)
        out.append(g if where is None else distribute_tensor(g, *meshes[where]))
    return out


def _rank(rank, world, path, name, out):
    dist.init_process_group("gloo", init_method=f"file://{path}", rank=rank, world_size=world,
                            timeout=datetime.timedelta(seconds=20))
    norms = []

    def norm(grads):
        norms.append(clip.sharded_norm(grads))
        return norms[-1]

    clip._Batch, clip._check_device, optimizer.sharded_norm = _Batch, lambda g: None, norm
    try:
        grads = _grads(name, world)
        params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
        for p, g in zip(params, grads):
            p.grad = g
        opt = LUMA(params, max_grad_norm=0.5)
        for _ in range(2):
            if any(opt._unwrap_tensor(p).numel() for p in params):
                with pytest.raises(RuntimeError, match="ROCm GPU"):
                    opt.step()
            else:
                opt.step()
                assert opt.grad_norm == norms[-1]
        want = sum(float(((g.full_tensor() if hasattr(g, "full_tensor") else g).double() ** 2)
                         .sum()) for g in grads) ** 0.5
        out[rank] = (want, [float(n) for n in norms])
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("name", SETS)
def test_ranks_join_the_same_reductions(name, tmp_path):
    with mp.Manager() as m:
        out = m.dict()
        mp.spawn(_rank, args=(2, str(tmp_path / "rdv"), name, out), nprocs=2)
        for rank in range(2):
            want, norms = out[rank]
            assert len(norms) == 2
            assert all(abs(n - want) <= 2.0 ** -23 * want for n in norms)
