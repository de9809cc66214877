"""The norm of nothing, with and without the host module."""

import pytest
import torch

import luma_amd


@pytest.mark.parametrize("module", [True, False])
def test_no_tensors(module, monkeypatch):
    if not module:
        monkeypatch.setattr(luma_amd.clip, "_host", lambda: None)
    p = torch.nn.Parameter(torch.ones(3))
    for total in (luma_amd.get_total_norm([]), luma_amd.clip_grad_norm_([], 1.0),
                  luma_amd.clip_grad_norm_([p], 1.0),
                  luma_amd.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)):
        assert total.dim() == 0 and total.dtype == torch.float32 and float(total) == 0.0
    luma_amd.clip_grads_with_norm_([p], 1.0, torch.tensor(2.0))
