"""linear_cross_entropy: what can be checked without a GPU (arguments, the
library's refusals and workspace sizes)."""

import ctypes
import re

import pytest
import torch

from luma_amd import _lib as L
from luma_amd import linear_cross_entropy


def _args(**change):
    """Arguments that only the library's own checks look at (nothing is launched)."""
    a = dict(hidden=256, weight=256, target=256, n=100, h=64, v=300, ld_hidden=64, ld_weight=64,
             ignore_index=-100, dtype=L.GRAD_BF16, reduction=L.XENT_MEAN, loss=256, stats=256,
             grad_loss=256, d_hidden=256, d_weight=256)
    a.update(change)
    return L.XentArgs(**a)


@pytest.mark.parametrize("change,text", [
    (dict(n=0), "empty"), (dict(h=0), "empty"), (dict(v=-1), "empty"),
    (dict(n=1 << 31), "too large"), (dict(h=1 << 21, ld_hidden=1 << 21, ld_weight=1 << 21), "too large"),
    (dict(n=1 << 24, v=1 << 24), "too large"), (dict(n=1 << 20, v=1 << 20), "too large"),
    (dict(dtype=3), "type"), (dict(dtype=-1), "type"), (dict(reduction=3), "reduction"),
    (dict(hidden=None), "null"), (dict(weight=None), "null"), (dict(target=None), "null"),
    (dict(stats=None), "null"), (dict(loss=None), "null"), (dict(ld_hidden=63), "overlap"),
    (dict(ld_weight=63), "overlap"), (dict(ld_weight=1 << 22), "too far apart")])
def test_library_refuses(change, text):
    lib = L.load()
    args = _args(**change)
    assert lib.luma_xent_workspace_bytes(ctypes.byref(args), 0) == -1
    assert re.search(text, lib.luma_last_error().decode())
    assert lib.luma_xent_forward(ctypes.byref(args), None) != 0


def test_workspace_is_checked():
    lib = L.load()
    for backward, name in ((0, "luma_xent_forward"), (1, "luma_xent_backward")):
        args = _args()
        size = lib.luma_xent_workspace_bytes(ctypes.byref(args), backward)
        assert size > 0
        for at, given in ((None, size), (256, size - 1), (264, size)):
            args.workspace, args.workspace_bytes = at, given
            assert getattr(lib, name)(ctypes.byref(args), None) != 0
            assert "workspace" in lib.luma_last_error().decode()
    assert lib.luma_xent_backward(ctypes.byref(_args(grad_loss=None)), None) != 0


def test_workspace_does_not_hold_the_logits():
    """A 128,256-word head (2.1 GB of 16-bit logits for 8,192 tokens): the forward
    keeps 8 bytes per token and 256 words; the backward at most 1 GiB of D, the
    hidden states' float32 sums and those of d_weight's last tiles."""
    lib = L.load()
    for n in (8192, 4 * 8192):
        args = _args(n=n, h=4096, v=128256, ld_hidden=4096, ld_weight=4096)
        size = lib.luma_xent_workspace_bytes(ctypes.byref(args), 0)
        assert size <= 8 * n * 501 + 64 * n
        size = lib.luma_xent_workspace_bytes(ctypes.byref(args), 1)
        assert size <= (1 << 30) + 4 * n * 4096 + (256 << 20)


def test_layout():
    assert ctypes.sizeof(L.XentArgs) == 136


def test_arguments():
    x, w, t = torch.ones(4, 8), torch.ones(6, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, t, reduction="max")
    with pytest.raises(ValueError, match="do not match"):
        linear_cross_entropy(x[:, :4], w, t)
    with pytest.raises(ValueError, match="int64"):
        linear_cross_entropy(x, w, t.int())
    with pytest.raises(ValueError, match="dtype"):
        linear_cross_entropy(x.double(), w.double(), t)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        linear_cross_entropy(x, w, t)
