"""Gradient norm and clipping: what can be checked without a GPU (arguments,
the library's refusals, the host module's table, the sum over shards)."""

import ctypes
import math
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import luma_amd
from luma_amd import _lib as L
from luma_amd import clip


def test_arguments_are_checked_first():
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match="norm_type"):
        luma_amd.clip_grad_norm_([p], 1.0, 3.0)
    with pytest.raises(ValueError, match="max_norm"):
        luma_amd.clip_grad_norm_([p], -1.0)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        luma_amd.clip_grad_norm_([p], 1.0)
    assert torch.equal(p.grad, torch.ones(3))


@pytest.mark.parametrize("shape,stride,dense", [
    ((3, 4), (4, 1), True), ((3, 4), (1, 3), True), ((3, 4), (8, 1), False),
    ((3, 1, 4), (4, 99, 1), True), ((5,), (2,), False), ((5,), (0,), False),
    ((2, 3, 4, 5), (60, 1, 15, 3), True), ((0, 7), (7, 1), True), ((), (), True)])
def test_dense(shape, stride, dense):
    t = torch.empty(1000).as_strided(shape, stride)
    assert clip._is_dense(t) is dense


def test_rows_add_up_their_tiles():
    grads = [torch.empty(n) for n in (1, 2048, 2049, 5000)]
    rows = clip._rows(grads)
    assert rows["first_tile"].tolist() == [0, 1, 2, 4]
    assert rows["numel"].tolist() == [1, 2048, 2049, 5000]
    assert rows["data"].tolist() == [g.data_ptr() for g in grads]


def test_spans_that_touch_are_apart():
    flat = torch.empty(100)
    clip._check_apart([flat[50:], flat[:50]])
    with pytest.raises(ValueError, match="share memory"):
        clip._check_apart([flat[49:], flat[:50]])


def _args(**change):
    """Arguments that only the library's own checks look at (nothing is launched)."""
    rows = np.zeros(2, dtype=L.GRAD_DTYPE)
    rows["data"] = 64
    rows["numel"] = 3000
    rows["first_tile"] = [0, 2]
    for k in ("data", "numel", "dtype", "first_tile"):
        if k in change:
            rows[k] = change.pop(k)
    a = dict(grads=rows.ctypes.data, n=2, norm=L.NORM_L2, max_norm=1.0, partials=64, total=64)
    a.update(change)
    return rows, L.NormArgs(**a)


@pytest.mark.parametrize("change,text", [
    (dict(grads=None), "null"), (dict(n=0), "no rows"), (dict(n=-1), "no rows"),
    (dict(norm=3), "unknown norm"), (dict(numel=[3000, 0]), "empty row"),
    (dict(data=[0, 64]), "empty row"), (dict(dtype=[0, 3]), "type"),
    (dict(first_tile=[0, 1]), "add up"), (dict(numel=[1 << 50, 1]), "too many"),
    (dict(n=1 << 20), "without a device table"), (dict(total=None), "null|no output"),
    (dict(partials=None), "null"), (dict(max_norm=-1.0), "max_norm"),
    (dict(max_norm=math.nan), "max_norm")])
def test_library_refuses(change, text):
    lib = L.load()
    rows, args = _args(**change)
    assert lib.luma_grad_clip(ctypes.byref(args), None) != 0
    import re
    assert re.search(text, lib.luma_last_error().decode())


def test_library_layout():
    assert L.GRAD_DTYPE.itemsize == 24 and ctypes.sizeof(L.NormArgs) == 72
    header = open(os.path.join(os.path.dirname(L.HERE), "include", "luma.h")).read()
    for name in ("GRAD_TILE", "GRADS_INLINE", "NORM_PARTIALS", "NORM_L2", "NORM_L1", "NORM_INF"):
        assert f"#define LUMA_{name} {getattr(L, name)}\n" in header


def test_host_module_leaves_what_it_cannot_take():
    host = L.load_host()
    if host is None:
        pytest.skip("the host module is not built")
    rows = np.zeros(1, dtype=L.GRAD_DTYPE)
    at = rows.ctypes.data
    assert host.grad_rows([], True, True, at) == (0, -1)
    p = torch.nn.Parameter(torch.ones(3))
    assert host.grad_rows([p], True, True, at) == (0, -1)      # no gradient
    p.grad = torch.ones(3)
    assert host.grad_rows([p], True, True, at) is None           # not on a GPU
    assert host.grad_rows([3], True, True, at) is None


def _join(rank, world, path, out):
    dist.init_process_group("gloo", init_method=f"file://{path}", rank=rank, world_size=world)
    from torch.distributed.device_mesh import init_device_mesh
    mesh = init_device_mesh("cpu", (world,))
    power = torch.tensor(float(3 + rank), dtype=torch.float64)
    top = power.clone()
    clip._join_shards(power, L.NORM_L2, mesh, (0,))
    clip._join_shards(top, L.NORM_INF, mesh, (0,))
    out[rank] = (float(power), float(top))
    dist.destroy_process_group()


def test_shards_of_two_ranks(tmp_path):
    with mp.Manager() as m:
        out = m.dict()
        mp.spawn(_join, args=(2, str(tmp_path / "rdv"), out), nprocs=2)
        assert dict(out) == {0: (7.0, 4.0), 1: (7.0, 4.0)}


def test_placements():
    from torch.distributed.tensor import Partial, Replicate, Shard

    class T:
        def __init__(self, *placements):
            self.placements = placements

    assert clip._shard_dims(T(Replicate(), Shard(1))) == (1,)
    assert clip._shard_dims(T(Shard(0), Shard(0))) == (0, 1)
    assert clip._shard_dims(T(Replicate())) == ()
    with pytest.raises(ValueError, match="Partial"):
        clip._shard_dims(T(Partial()))
