"""examples/train_lm.py with dropout: it runs, its masks follow from the steps'
numbers, and its model's gradients are those of the same model of torch's layers."""

import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

import luma_amd

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "train_lm.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_lm", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_it_runs_and_repeats(example):
    runs = [example.train(8, vocab=300, width=48, layers=2, batch=8, length=16, every=0, dropout=0.2)
            for _ in range(2)]
    assert bool(runs[0].isfinite().all()) and runs[0].shape == (8,)
    assert torch.equal(runs[0][:1], runs[1][:1])
    plain = example.train(1, vocab=300, width=48, layers=2, batch=8, length=16, every=0)
    assert float(plain[0]) != float(runs[0][0])


def test_gradients_of_its_model(example):
    """Without dropout, float32, against the same formulas of torch's layers in 64 bits:
    relative to each gradient 1e-5, some hundred roundings of 2^-24."""
    torch.manual_seed(3)
    model = example.Model(200, 48, 2).cuda()
    words = torch.randint(0, 200, (6, 17), device="cuda")
    loss = luma_amd.linear_cross_entropy(model(words[:, :-1]), model.embed.weight, words[:, 1:])
    got = torch.autograd.grad(loss, list(model.parameters()))
    exact = example.Model(200, 48, 2).cuda().double()
    exact.load_state_dict({k: v.double() for k, v in model.state_dict().items()})
    x = exact.embed(words[:, :-1])
    count = torch.arange(1, 17, device="cuda")[:, None]
    for i, (mix, up, down) in enumerate(zip(exact.mix, exact.up, exact.down)):
        y = exact.norm[2 * i](x)
        x = x + mix(torch.cat([y, y.cumsum(1) / count], dim=-1))
        x = x + down(F.gelu(up(exact.norm[2 * i + 1](x))))
    logits = (exact.norm[-1](x) @ exact.embed.weight.T).flatten(0, 1)
    want = torch.autograd.grad(F.cross_entropy(logits, words[:, 1:].flatten()),
                               list(exact.parameters()))
    for p, q in zip(got, want):
        assert float((p.double() - q).norm()) <= 1e-5 * float(q.norm())
