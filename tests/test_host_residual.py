"""layer_norm, add_layer_norm and dropout: what can be checked without a GPU
(arguments, the library's refusals and workspace sizes, the draws' definition)."""

import ctypes
import re

import numpy as np
import pytest
import torch

import residual_util
from luma_amd import _lib as L
from luma_amd import add_layer_norm, dropout, layer_norm


def _norm_args(**change):
    """Arguments that only the library's own checks look at (nothing is launched)."""
    a = dict(x=256, weight=256, bias=256, n=100, h=64, ld_x=64, ld_residual=64, stream=L.GRAD_BF16,
             branch=L.GRAD_BF16, param=L.GRAD_F32, eps=1e-5, y=256, stats=256, d_y=256, d_x=256,
             d_weight=256, d_bias=256)
    a.update(change)
    return L.LayerNormArgs(**a)


def _refused(name, args, text):
    lib = L.load()
    assert getattr(lib, name)(ctypes.byref(args), None) != 0
    assert re.search(text, lib.luma_last_error().decode())


@pytest.mark.parametrize("change,text", [
    (dict(n=0), "empty"), (dict(h=0), "empty"), (dict(n=-1), "empty"), (dict(n=1 << 31), "large"),
    (dict(h=(1 << 24) + 1), "large"), (dict(stream=3), "type"), (dict(branch=-1), "type"),
    (dict(stream=L.GRAD_F16), "stream"), (dict(branch=L.GRAD_F32), "stream"),
    (dict(param=L.GRAD_F16), "weight"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(reserved=1), "reserved"), (dict(drop=L.Dropout(p=0.1)), "residual"),
    (dict(drop=L.Dropout(p=1.5)), "dropped"), (dict(drop=L.Dropout(p=float("nan"))), "dropped")])
def test_norm_refuses(change, text):
    _refused("luma_layer_norm_forward", _norm_args(**change), text)
    _refused("luma_layer_norm_backward", _norm_args(**change), text)


@pytest.mark.parametrize("name,change,text", [
    ("forward", dict(x=None), "null"), ("forward", dict(y=None), "null"),
    ("forward", dict(residual=256), "null"), ("forward", dict(ld_x=-64), "backwards"),
    ("forward", dict(residual=256, total=256, ld_residual=-1), "backwards"),
    ("backward", dict(x=None), "null"), ("backward", dict(d_y=None), "null"),
    ("backward", dict(ld_x=-64), "backwards"),
    ("backward", dict(stats=None), "null"), ("backward", dict(d_total=256), "without"),
    ("backward", dict(d_residual=256), "without"), ("backward", dict(), "workspace"),
    ("backward", dict(workspace=256, workspace_bytes=16), "workspace"),
    ("backward", dict(workspace=264, workspace_bytes=1 << 40), "workspace")])
def test_norm_refuses_one_way(name, change, text):
    _refused(f"luma_layer_norm_{name}", _norm_args(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(numel=0), "empty"),
    (dict(numel=(1 << 36) + 1), "large"), (dict(in_type=3), "types"),
    (dict(in_type=L.GRAD_F16), "types"), (dict(drop=L.Dropout(p=-0.1)), "dropped"),
    (dict(drop=L.Dropout(p=0.5, reserved=1)), "reserved")])
def test_dropout_refuses(change, text):
    a = dict(x=256, y=256, numel=100, in_type=L.GRAD_BF16, out_type=L.GRAD_BF16)
    a.update(change)
    _refused("luma_dropout", L.DropoutArgs(**a), text)


@pytest.mark.parametrize("numel", [(1 << 34) + 1, 1 << 35, 1 << 36])
@pytest.mark.parametrize("in_type,out_type", [(L.GRAD_F32, L.GRAD_F32), (L.GRAD_BF16, L.GRAD_BF16),
                                              (L.GRAD_F16, L.GRAD_F32)])
def test_dropout_refuses_more_than_a_launch(numel, in_type, out_type):
    """2,048 or 4,096 elements a workgroup of 256: more than 2^34 could be 2^32
    threads, which no launch has."""
    a = L.DropoutArgs(x=256, y=256, numel=numel, in_type=in_type, out_type=out_type)
    _refused("luma_dropout", a, "large")


@pytest.mark.parametrize("n,h", [(1, 1), (100, 64), (8192, 768), (16384, 4096), (10, 16384),
                                 (10, 16385), (3, 1 << 24), (1 << 30, 8)])
def test_workspace(n, h):
    """Two float32 sums a column for each workgroup that stays on the chip."""
    size = L.load().luma_layer_norm_workspace_bytes(ctypes.byref(_norm_args(n=n, h=h)))
    assert 8 * h <= size <= max(8 * h, 1024 * 8 * max(h, 1))
    assert size <= max(8 * h, 8 * h * n)


def test_null_arguments():
    lib = L.load()
    for name in ("luma_dropout", "luma_layer_norm_forward", "luma_layer_norm_backward"):
        assert getattr(lib, name)(None, None) != 0
    assert lib.luma_layer_norm_workspace_bytes(None) == -1


def test_draws_are_the_librarys_generator():
    counter = np.array([[0, 0, 0, 0], [7, 1, 1, 5], [0xFFFFFFFF, 3, 0, 0xFFFFFFFF]], np.uint64)
    key = (0x12345678, 0x9ABCDEF0)
    got = residual_util.philox(counter, key)
    for c, words in zip(counter, got):
        assert L.philox4x32(c, key) == [int(w) for w in words]


def test_arguments():
    x, w = torch.ones(4, 8), torch.ones(8)
    with pytest.raises(ValueError, match="p must be"):
        dropout(x, 1.5, 0)
    with pytest.raises(ValueError, match="p must be"):
        dropout(x, float("nan"), 0)
    with pytest.raises(ValueError, match="call must be"):
        dropout(x, 0.5, 0, -1)
    with pytest.raises(ValueError, match="seed must fit"):
        dropout(x, 0.5, 1 << 64)
    with pytest.raises(ValueError, match="int64"):
        dropout(x, 0.5, torch.zeros(1))
    with pytest.raises(ValueError, match="one int64"):
        dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="not float32/bfloat16/float16"):
        dropout(x.double(), 0.5, 0)
    with pytest.raises(ValueError, match="do not match"):
        dropout(x, 0.5, 0, residual=x[:2])
    with pytest.raises(ValueError, match="residual is"):
        dropout(x, 0.5, 0, residual=x.half())
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        dropout(x, 0.5, 0)
    with pytest.raises(ValueError, match="not float32/bfloat16/float16"):
        layer_norm(x.double())
    with pytest.raises(ValueError, match="not float32/bfloat16/float16"):
        layer_norm(x, dtype=torch.float64)
    with pytest.raises(ValueError, match="a result from"):
        layer_norm(x.half(), dtype=torch.float32)
    with pytest.raises(ValueError, match="no rows"):
        layer_norm(torch.tensor(1.0))
    with pytest.raises(ValueError, match="no rows"):
        layer_norm(x[:, :0])
    with pytest.raises(ValueError, match="do not match"):
        layer_norm(x, w[:4])
    with pytest.raises(ValueError, match="weight is"):
        layer_norm(x, w.half())
    with pytest.raises(ValueError, match="bias"):
        layer_norm(x.half(), w.half(), w)
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, eps=-1.0)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        layer_norm(x, w, w)
    with pytest.raises(ValueError, match="residual"):
        add_layer_norm(x, x[:2])
    with pytest.raises(ValueError, match="residual is"):
        add_layer_norm(x.half(), x.bfloat16())
    with pytest.raises(ValueError, match="p must be"):
        add_layer_norm(x, x, p=-0.5)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        add_layer_norm(x, x, w, w)


def test_layout():
    assert [ctypes.sizeof(t) for t in (L.Dropout, L.DropoutArgs, L.LayerNormArgs)] == [32, 72, 208]
