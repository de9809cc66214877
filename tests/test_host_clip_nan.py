"""The largest gradient of all shards: a NaN or an infinity on any rank is every
rank's."""

import math

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from luma_amd import _lib as L
from luma_amd import clip

CASES = [(math.nan, 2.0, 1.0), (2.0, math.nan, 1.0), (2.0, 1.0, math.nan), (math.nan,) * 3,
         (math.inf, math.nan, 0.0), (math.nan, 0.0, math.inf), (1.0, math.inf, 2.0),
         (0.0, 3e-42, 0.0), (5.0, 7.0, 6.0)]


def _rank(rank, world, path, out):
    from torch.distributed.device_mesh import init_device_mesh
    dist.init_process_group("gloo", init_method=f"file://{path}", rank=rank, world_size=world)
    try:
        mesh = init_device_mesh("cpu", (world,))
        got = []
        for case in CASES:
            power = torch.tensor(case[rank], dtype=torch.float64)
            clip._join_shards(power, L.NORM_INF, mesh, (0,))
            got.append(float(power))
        out[rank] = got
    finally:
        dist.destroy_process_group()


def test_three_ranks(tmp_path):
    with mp.Manager() as m:
        out = m.dict()
        mp.spawn(_rank, args=(3, str(tmp_path / "rdv"), out), nprocs=3)
        for rank in range(3):
            for case, got in zip(CASES, out[rank]):
                if any(map(math.isnan, case)):
                    assert math.isnan(got), (rank, case, got)
                else:
                    assert got == max(case), (rank, case, got)
