"""examples/train_lm.py: loss, gradient norm, clipping and step together."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "train_lm.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_lm", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_it_learns_by_either_clipping(example):
    """The loss starts at that of a uniform guess (log 1000 = 6.9) and falls; the
    first step of both ways of clipping starts from the same weights."""
    runs = [example.train(60, vocab=1000, width=64, layers=1, batch=16, length=32, clip=clip,
                          every=0) for clip in ("step", "before")]
    for losses in runs:
        assert bool(losses.isfinite().all())
        assert 6.4 < float(losses[0]) < 7.4
        assert float(losses[-5:].mean()) < float(losses[0]) - 0.5
    assert torch.equal(runs[0][0], runs[1][0])
    assert abs(float(runs[0][-1]) - float(runs[1][-1])) < 0.2
