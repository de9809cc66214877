"""policy_loss: what can be checked without a GPU (arguments, the library's
refusals and workspace sizes)."""

import ctypes
import re

import pytest
import torch

from luma_amd import _lib as L
from luma_amd import policy_loss


def _args(**change):
    """Arguments that only the library's own checks look at (nothing is launched)."""
    a = dict(logp=256, old_logp=256, ref_logp=256, advantage=256, mask=256, rows=100, length=640,
             ld_logp=640, ld_old=640, ld_ref=640, ld_advantage=1, ld_mask=640, dtype=L.GRAD_F32,
             reduction=L.XENT_MEAN, clip_low=0.2, clip_high=0.2, kl_weight=0.1, loss=256, stats=256,
             share=256, grad_loss=256, d_logp=256)
    a.update(change)
    return L.PolicyArgs(**a)


@pytest.mark.parametrize("change,text", [
    (dict(rows=0), "empty"), (dict(length=-1), "empty"), (dict(rows=1 << 31), "large"),
    (dict(length=1 << 31), "large"), (dict(rows=1 << 30, length=1 << 20), "large"),
    (dict(rows=(1 << 22) + 1, length=2000), "large"), (dict(dtype=3), "type"),
    (dict(reduction=4), "reduction"), (dict(reduction=-1), "reduction"),
    (dict(clip_low=-0.1), "clip_low"), (dict(clip_low=1.1), "clip_low"),
    (dict(clip_low=float("nan")), "clip_low"), (dict(clip_high=-0.1), "clip_high"),
    (dict(kl_weight=float("nan")), "kl_weight"), (dict(reserved=1), "reserved"),
    (dict(logp=None), "null"), (dict(old_logp=None), "null"), (dict(advantage=None), "null"),
    (dict(ld_logp=-1), "backwards"), (dict(ld_mask=-1), "backwards"),
    (dict(ld_ref=-1), "backwards")])
def test_library_refuses(change, text):
    lib = L.load()
    args = _args(**change)
    assert lib.luma_policy_workspace_bytes(ctypes.byref(args)) == -1
    assert re.search(text, lib.luma_last_error().decode())
    assert lib.luma_policy_forward(ctypes.byref(args), None) != 0
    assert lib.luma_policy_backward(ctypes.byref(args), None) != 0


def test_library_refuses_one_way():
    lib = L.load()
    for name, change, text in (("forward", dict(loss=None), "null"),
                               ("forward", dict(), "workspace"),
                               ("forward", dict(workspace=256, workspace_bytes=16), "workspace"),
                               ("forward", dict(workspace=264, workspace_bytes=1 << 30), "workspace"),
                               ("backward", dict(grad_loss=None), "null"),
                               ("backward", dict(share=None), "null"),
                               ("backward", dict(d_logp=None), "null")):
        assert getattr(lib, f"luma_policy_{name}")(ctypes.byref(_args(**change)), None) != 0
        assert re.search(text, lib.luma_last_error().decode())
    assert lib.luma_policy_forward(None, None) != 0
    assert lib.luma_policy_backward(None, None) != 0
    assert lib.luma_policy_workspace_bytes(None) == -1


@pytest.mark.parametrize("rows,length", [(1, 1), (100, 640), (1 << 20, 1000), (1, 1 << 30),
                                         (512, 8192), (1 << 22, 1025), (3, 1 << 20)])
def test_workspace(rows, length):
    """A record of 48 bytes for each workgroup, and not for each token."""
    size = L.load().luma_policy_workspace_bytes(ctypes.byref(_args(rows=rows, length=length)))
    assert 0 <= size <= 48 * max(rows, 4100)


def test_arguments():
    lp, a = torch.zeros(4, 8), torch.zeros(4)
    with pytest.raises(ValueError, match="reduction"):
        policy_loss(lp, lp, a, reduction="max")
    for change in (dict(clip_low=-0.1), dict(clip_low=1.5), dict(clip_high=-1.0),
                   dict(kl_weight=float("nan")), dict(clip_high=float("nan"))):
        with pytest.raises(ValueError, match="clip_low must be"):
            policy_loss(lp, lp, a, **change)
    with pytest.raises(ValueError, match="not float32"):
        policy_loss(lp.double(), lp.double(), a)
    with pytest.raises(ValueError, match="no dimension"):
        policy_loss(a[0], a[0], a[0])
    with pytest.raises(ValueError, match="old_logp torch.float16"):
        policy_loss(lp, lp.half(), a)
    with pytest.raises(ValueError, match="old_logp"):
        policy_loss(lp, lp[:, :4], a)
    with pytest.raises(ValueError, match="ref_logp"):
        policy_loss(lp, lp, a, ref_logp=lp[:2])
    with pytest.raises(ValueError, match="mask must be bool"):
        policy_loss(lp, lp, a, lp)
    with pytest.raises(ValueError, match="mask"):
        policy_loss(lp, lp, a, lp[:2] > 0)
    with pytest.raises(ValueError, match="advantage must be float32"):
        policy_loss(lp, lp, a.half())
    with pytest.raises(ValueError, match="advantage"):
        policy_loss(lp, lp, a[:2])
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        policy_loss(lp, lp, a)


def test_layout():
    assert ctypes.sizeof(L.PolicyArgs) == 192
