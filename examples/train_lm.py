"""Trains a small language model with the framework's operators: layer norms,
each in one kernel with the sum before it (and its dropout), the loss over the
vocabulary without its logits, the gradients' norm and clipping, and the LUMA
step.

    python examples/train_lm.py [--steps 300] [--vocab 8192] [--clip step|before] [--dropout 0.1]

``--clip step`` gives the optimizer ``max_grad_norm``: the norm is taken and
the gradients are clipped inside ``step()``, as its kernels read them.
``--clip before`` calls ``luma_amd.clip_grad_norm_`` between ``backward()`` and
``step()``, as the reference's benchmark does with torch's
(benchmarks/bench_nanogpt.py).  Dropout's masks follow from a step's number and
are drawn again in the backward.  The text is synthetic: a random walk over the
words, each with a few likely successors.
"""

import argparse
import os
import sys
import time

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import luma_amd  # noqa: E402


class Model(nn.Module):
    """Embeddings, causal averages of the words before and MLPs; the head is
    the embedding's weight.  ``forward`` gives the last hidden states.  The
    residual stream is float32, the branches are of autocast's type."""

    def __init__(self, vocab, width, layers):
        super().__init__()
        self.embed = nn.Embedding(vocab, width)
        self.mix = nn.ModuleList(nn.Linear(2 * width, width) for _ in range(layers))
        self.up = nn.ModuleList(nn.Linear(width, 4 * width) for _ in range(layers))
        self.down = nn.ModuleList(nn.Linear(4 * width, width) for _ in range(layers))
        self.norm = nn.ModuleList(nn.LayerNorm(width) for _ in range(2 * layers + 1))
        nn.init.normal_(self.embed.weight, std=0.02)

    def forward(self, words, dropout=0.0, seed=0):
        x = self.embed(words)
        count = torch.arange(1, words.shape[1] + 1, device=words.device)[:, None]
        kind = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else None
        borders = iter(enumerate(self.norm))

        def border(branch, x):
            """x with a branch's output, and what the next branch reads."""
            call, norm = next(borders)
            if branch is None:
                return luma_amd.layer_norm(x, norm.weight, norm.bias, norm.eps, dtype=kind), x
            return luma_amd.add_layer_norm(branch, x, norm.weight, norm.bias, norm.eps, p=dropout,
                                           seed=seed, call=call)

        y, x = border(None, x)
        for mix, up, down in zip(self.mix, self.up, self.down):
            y, x = border(mix(torch.cat([y, y.cumsum(1) / count], dim=-1)), x)
            y, x = border(down(F.gelu(up(y))), x)
        return y


def text(vocab, batch, length, generator, successors):
    """A batch of random walks over `successors` [vocab][k]."""
    words = torch.empty((batch, length), dtype=torch.int64, device=successors.device)
    words[:, 0] = torch.randint(vocab, (batch,), generator=generator, device=words.device)
    for i in range(1, length):
        pick = torch.randint(successors.shape[1], (batch,), generator=generator,
                             device=words.device)
        words[:, i] = successors[words[:, i - 1], pick]
    return words


def train(steps=300, vocab=8192, width=256, layers=2, batch=32, length=64, clip="step",
          max_norm=0.5, lr=2e-3, seed=0, every=50, say=print, dropout=0.0):
    """Runs `steps` steps; the losses."""
    torch.manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    successors = torch.randint(vocab, (vocab, 4), generator=gen, device="cuda")
    model = Model(vocab, width, layers).cuda()
    params = list(model.parameters())
    opt = luma_amd.LUMA(params, lr=lr, weight_decay=0.01,
                        max_grad_norm=max_norm if clip == "step" else None)
    losses, began = [], time.perf_counter()
    for step in range(steps):
        words = text(vocab, batch, length + 1, gen, successors)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            hidden = model(words[:, :-1], dropout, seed=step)
            loss = luma_amd.linear_cross_entropy(hidden, model.embed.weight, words[:, 1:])
        opt.zero_grad()
        loss.backward()
        norm = (luma_amd.clip_grad_norm_(params, max_norm) if clip == "before" else None)
        opt.step()
        losses.append(loss.detach())
        if every and step % every == 0:
            norm = opt.grad_norm if norm is None else norm
            say(f"step {step:5d}  loss {float(losses[-1]):.4f}  gradient norm {float(norm):.3f}")
    torch.cuda.synchronize()
    if every:
        rate = steps * batch * length / (time.perf_counter() - began)
        say(f"{steps} steps, loss {float(losses[-1]):.4f}, {rate:.0f} words/s")
    return torch.stack(losses)


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--steps", type=int, default=300)
    parser.add_argument("--vocab", type=int, default=8192)
    parser.add_argument("--clip", choices=("step", "before"), default="step")
    parser.add_argument("--dropout", type=float, default=0.0)
    args = parser.parse_args()
    train(args.steps, args.vocab, clip=args.clip, dropout=args.dropout)
