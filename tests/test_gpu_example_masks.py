"""examples/train_lm.py's dropout: its masks follow from the step's number and the
border's place, and its model's gradients are those of the same masks in 64 bits."""

import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

import luma_amd
import residual_util

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "train_lm.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_lm", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_seeds_and_calls(example, monkeypatch):
    """Each step has its own seed, and each border of a step its own call."""
    seen, real = [], luma_amd.add_layer_norm

    def record(*args, p=0.0, seed=0, call=0):
        seen.append((p, seed, call))
        return real(*args, p=p, seed=seed, call=call)

    monkeypatch.setattr(luma_amd, "add_layer_norm", record)
    example.train(3, vocab=300, width=48, layers=2, batch=8, length=16, every=0, dropout=0.2)
    assert len(seen) == 3 * 4 and len(set(seen)) == len(seen)
    for step in range(3):
        part = seen[4 * step:4 * step + 4]
        assert all((p, seed) == (0.2, step) for p, seed, _ in part)
        assert len({call for _, _, call in part}) == 4


def test_outputs_follow_from_the_seed(example):
    torch.manual_seed(1)
    model = example.Model(200, 48, 2).cuda()
    words = torch.randint(0, 200, (6, 16), device="cuda")
    with torch.no_grad():
        first, again, other = (model(words, 0.3, seed=s) for s in (0, 0, 1))
    assert torch.equal(first, again) and not torch.equal(first, other)


def test_gradients_with_dropout(example):
    """Float32 against the same formulas in 64 bits with the masks of the draws'
    definition: relative to each gradient 1e-5, some hundred roundings of 2^-24."""
    torch.manual_seed(3)
    p, seed = 0.25, 12
    model = example.Model(200, 48, 2).cuda()
    words = torch.randint(0, 200, (6, 17), device="cuda")
    hidden = model(words[:, :-1], p, seed=seed)
    loss = luma_amd.linear_cross_entropy(hidden, model.embed.weight, words[:, 1:])
    got = torch.autograd.grad(loss, list(model.parameters()))
    exact = example.Model(200, 48, 2).cuda().double()
    exact.load_state_dict({k: v.double() for k, v in model.state_dict().items()})
    x = exact.embed(words[:, :-1])
    count = torch.arange(1, 17, device="cuda")[:, None]

    def kept(call):
        return residual_util.kept((6, 16, 48), p, seed, call).cuda() / (1 - p)

    for i, (mix, up, down) in enumerate(zip(exact.mix, exact.up, exact.down)):
        y = exact.norm[2 * i](x)
        x = x + mix(torch.cat([y, y.cumsum(1) / count], dim=-1)) * kept(2 * i + 1)
        x = x + down(F.gelu(up(exact.norm[2 * i + 1](x)))) * kept(2 * i + 2)
    logits = (exact.norm[-1](x) @ exact.embed.weight.T).flatten(0, 1)
    want = torch.autograd.grad(F.cross_entropy(logits, words[:, 1:].flatten()),
                               list(exact.parameters()))
    for a, b in zip(got, want):
        assert float((a.double() - b).norm()) <= 1e-5 * float(b.norm())
