"""Gradients without elements: their norm is a 0 on their device, as the norm
of any gradients is, by every path."""

import pytest
import torch

import luma_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("module", [True, False])
@pytest.mark.parametrize("count", [1, 3, 700])
def test_norm_lies_on_the_device(count, module, monkeypatch):
    if not module:
        monkeypatch.setattr(luma_amd.clip, "_host", lambda: None)
    params = [torch.nn.Parameter(torch.empty((0, 7), device="cuda")) for _ in range(count)]
    for p in params:
        p.grad = torch.empty_like(p)
    for total in (luma_amd.get_total_norm([p.grad for p in params]),
                  luma_amd.clip_grad_norm_(params, 1.0),
                  luma_amd.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)):
        assert total.is_cuda and total.dim() == 0 and total.dtype == torch.float32
        assert float(total) == 0.0
    luma_amd.clip_grads_with_norm_(params, 1.0, torch.tensor(2.0))
