"""Which of a DTensor gradient's mesh dimensions its norm is summed over."""

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
from torch.distributed.tensor import Partial, Replicate, Shard
from torch.distributed.tensor.placement_types import _StridedShard

from luma_amd import _lib as L
from luma_amd import clip


class _T:
    def __init__(self, *placements):
        self.placements = placements


@pytest.mark.parametrize("placements,dims", [
    ((_StridedShard(0, split_factor=2), Shard(0)), (0, 1)),   # fully_shard of a tensor-parallel weight
    ((Replicate(), _StridedShard(0, split_factor=2), Shard(0)), (1, 2)),
    ((_StridedShard(1, split_factor=4), Replicate()), (0,)),
    ((Shard(1), Replicate(), Shard(0)), (0, 2))])
def test_every_spread_dimension_counts(placements, dims):
    assert clip._shard_dims(_T(*placements)) == dims


def test_partial_is_refused_beside_a_strided_shard():
    with pytest.raises(ValueError, match="Partial"):
        clip._shard_dims(_T(_StridedShard(0, split_factor=2), Partial()))


class _Batch(clip._Batch):
    def args(self, norm, max_norm, total, power=None):
        return power

    def call(self, name, power):
        for g in self.hold:
            power += (g.double() ** 2).sum()


def _rank(rank, world, path, out):
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import DTensor
    dist.init_process_group("gloo", init_method=f"file://{path}", rank=rank, world_size=world)
    try:
        clip._Batch, clip._check_device = _Batch, lambda g: None
        mesh = init_device_mesh("cpu", (world, 1))
        local = torch.full((3, 2), 1.0 + rank)
        g = DTensor.from_local(local, mesh, [_StridedShard(0, split_factor=1), Shard(0)])
        out[rank] = float(clip.sharded_norm([g]))
    finally:
        dist.destroy_process_group()


def test_two_ranks_of_a_strided_shard(tmp_path):
    """6 (1 + 4) = 30 in all."""
    with mp.Manager() as m:
        out = m.dict()
        mp.spawn(_rank, args=(2, str(tmp_path / "rdv"), out), nprocs=2)
        for rank in range(2):
            assert abs(out[rank] ** 2 - 30.0) <= 30.0 * 2.0 ** -22
