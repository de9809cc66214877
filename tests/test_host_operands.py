"""The operators' refusals of operands that do not fit each other, without a GPU: the
operators' own code on host tensors, up to the library's checks."""

import ctypes

import pytest
import torch

import operands_util
from luma_amd import _lib as L
from luma_amd import loss, policy, residual

# (a call that nothing refused would launch a kernel on host memory)
pytestmark = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="for machines without a GPU")

CODE = {"dropout": residual._dropout_op, "dropout_backward": residual._dropout_backward_op,
        "layer_norm": residual._norm_op, "layer_norm_backward": residual._norm_backward_op,
        "policy_loss": policy._forward_op, "policy_loss_backward": policy._backward_op,
        "linear_cross_entropy": loss._forward_op,
        "linear_cross_entropy_backward": loss._backward_op}


class Launched(Exception):
    pass


@pytest.fixture(autouse=True)
def on_the_host(monkeypatch):
    def run(name, args, device):
        lib = L.load()
        if getattr(lib, name)(ctypes.byref(args), None) != 0:
            text = lib.luma_last_error().decode()
            # (a launch that failed for want of a device is one that was tried)
            raise Launched(text) if "device" in text or "HIP" in text else ValueError(text)
        raise Launched(name)

    monkeypatch.setattr(operands_util, "DEVICE", "cpu")
    for module in (residual, policy):
        monkeypatch.setattr(module, "_check_device", lambda *a, **k: None)
        monkeypatch.setattr(module, "_run", run)

    def call(name, args, device):
        size = L.load().luma_xent_workspace_bytes(ctypes.byref(args), name.endswith("backward"))
        if size < 0:
            L.check(-1, name)
        workspace = torch.empty(size + 256, dtype=torch.uint8)
        args.workspace, args.workspace_bytes = -(-workspace.data_ptr() // 256) * 256, size
        run(name, args, device)

    monkeypatch.setattr(loss, "_check", lambda *a, **k: None)
    monkeypatch.setattr(loss, "_call", call)


@pytest.mark.parametrize("name", operands_util.CALLS)
def test_what_fits(name):
    with pytest.raises(Launched):
        CODE[name]._init_fn(*operands_util.operands(name))


@pytest.mark.parametrize("name,change", [(n, c) for n, cs in operands_util.BAD.items() for c in cs])
def test_what_does_not_fit(name, change):
    with pytest.raises((ValueError, KeyError, L.LumaLibraryError)):
        CODE[name]._init_fn(*operands_util.operands(name, change))
