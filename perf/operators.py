"""The operators between a model's last hidden state and ``opt.step()``, as
cases to be timed and compared.

``loss`` is the cross entropy of a vocabulary's logits without the logits
being kept (``luma_amd.linear_cross_entropy``), ``grad`` the same with its
gradients for the hidden states and the vocabulary's weight; ``norm`` is the
global norm of many gradients (``luma_amd.get_total_norm``) and ``clip``
clipping them in place by it (``luma_amd.clip_grad_norm_``).

A case's fields: ``call``; for the loss ``tokens``, ``hidden``, ``vocab``,
``type``, ``reduction`` and ``ignored`` (the share of targets that are
``IGNORE``: padding, prompts); for the norm ``shapes`` and the fields that
name a list of shapes (``_shapes``), ``type``, ``std``, ``norm_type`` and
``packed`` (the gradients without padding between them, as in a bucket).
"""

import math
import random

import torch

own = False

DEV = "cuda"
IGNORE = -100
ALIGN = 64                     # elements: where a gradient of a flat buffer may start
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# -- the cases ------------------------------------------------------------------


def _loss(name, call, tokens, hidden, vocab, kind, reduction="mean", ignored=0.0):
    return {"name": name, "call": call, "tokens": tokens, "hidden": hidden, "vocab": vocab,
            "type": kind, "reduction": reduction, "ignored": ignored}


def _norm(name, call, shapes, kind="float32", norm_type=2.0, std=1e-3, **more):
    return dict({"name": name, "call": call, "shapes": shapes, "type": kind,
                 "norm_type": norm_type, "std": std}, **more)


def listed():
    return [
        # the nanoGPT-sized model's head (32 windows of 64 tokens, 28 characters): latency
        _loss("grad nano", "grad", 2048, 128, 28, "float32"),
        # scoring one token with the Llama-3-8B-shaped head: the weight is read once
        _loss("loss llama 1 token", "loss", 1, 4096, 128256, "bfloat16", "none"),
        # each token's loss with GPT-2 small's head, 8 windows of 1024 tokens: evaluation
        _loss("loss gpt2 bf16", "loss", 8192, 768, 50257, "bfloat16", "none"),
        # the same in a training step
        _loss("grad gpt2 bf16", "grad", 8192, 768, 50257, "bfloat16"),
        # a training step of the Llama-3-8B-shaped head: the largest
        _loss("grad llama bf16", "grad", 8192, 4096, 128256, "bfloat16"),
        # fine-tuning on answers: odd sizes, prompts ignored, each token's loss weighted
        _loss("grad ragged fp16", "grad", 1021, 1000, 32003, "float16", "none", 0.3),
        # GPT-2 small's head without mixed precision
        _loss("grad gpt2 fp32", "grad", 1024, 768, 50257, "float32"),
        # the nanoGPT-sized model (51 tensors, 0.8M parameters): launches and latency
        _norm("clip nano", "clip", "nano"),
        # GPT-2 small's gradients, an ordinary training step
        _norm("clip gpt2 bf16", "clip", "gpt2", "bfloat16"),
        # 20,000 tensors of 1 to 65,536 elements: many odd sizes in one call
        _norm("clip many small", "clip", "log_uniform", tensors=20000, most=65536, shape_seed=3),
        # the norm of the embeddings and 8 of 32 layers of the Llama-3-8B-shaped set, for a log
        _norm("norm llama bf16", "norm", "llama", "bfloat16", layers=8, embeddings=True),
        # the largest gradient, of odd-sized weights in a packed fp16 bucket
        _norm("norm packed fp16 inf", "norm", "log_uniform", "float16", math.inf, tensors=200,
              most=2000003, shape_seed=7, packed=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges."""
    call = rng.choice(["loss", "grad", "grad", "norm", "clip"])
    kind = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    if call in ("loss", "grad"):
        # (a float32 product costs many times a 16-bit one)
        most = 8192 * 4096 * 128256 // (16 if kind == "float32" else 1)
        n, h, v = (_log_uniform(rng, *r) for r in ((1, 8192), (64, 4096), (28, 131072)))
        if rng.random() < 0.5:
            h = max(64, h // 64 * 64)
        while n * h * v > most:
            n = (n + 1) // 2
        return {"call": call, "tokens": n, "hidden": h, "vocab": v, "type": kind,
                "reduction": rng.choice(["mean", "sum", "none"]),
                "ignored": rng.choice([0.0, 0.0, 0.3]) if n > 8 else 0.0}
    tensors = _log_uniform(rng, 1, 20000)
    most = _log_uniform(rng, 64, 1 << 26)
    while tensors * most > 1 << 30:
        most //= 2
    return {"call": call, "shapes": "log_uniform", "type": kind, "tensors": tensors, "most": most,
            "norm_type": rng.choice([2.0, 2.0, 1.0, math.inf]), "std": 10.0 ** rng.uniform(-4, -2),
            "shape_seed": rng.randrange(1 << 20), "packed": rng.random() < 0.5}


def _shapes(case):
    kind = case["shapes"]
    if kind == "nano":
        out = [(28, 128), (64, 128)]
        for _ in range(4):
            out += [(128,), (128,), (384, 128), (384,), (128, 128), (128,), (128,), (128,),
                    (512, 128), (512,), (128, 512), (128,)]
        return out + [(128,), (128,)]
    if kind == "gpt2":
        out = [(50257, 768), (1024, 768)]
        for _ in range(12):
            out += [(768,), (768,), (768, 2304), (2304,), (768, 768), (768,), (768,), (768,),
                    (768, 3072), (3072,), (3072, 768), (768,)]
        return out + [(768,), (768,)]
    if kind == "llama":
        out = [(128256, 4096)] if case["embeddings"] else []
        for _ in range(case["layers"]):
            out += [(4096, 4096), (1024, 4096), (1024, 4096), (4096, 4096), (14336, 4096),
                    (14336, 4096), (4096, 14336), (4096,), (4096,)]
        return out + ([(4096,), (128256, 4096)] if case["embeddings"] else [])
    rng = random.Random(case["shape_seed"])
    return [(_log_uniform(rng, 1, case["most"]),) for _ in range(case["tensors"])]


# -- inputs ---------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _head(case, seed):
    """Hidden states of a final norm, a head's weight, targets that are common
    words more often than rare ones, and the gradient of each token's loss (one
    for all but reduction "none").  The target's logit stands up to 12 over the
    others', as it comes to in training."""
    gen = _generator(seed)
    n, h, v = case["tokens"], case["hidden"], case["vocab"]
    weight = torch.randn((v, h), generator=gen, device=DEV).mul_(0.02)
    target = (torch.rand(n, generator=gen, device=DEV) ** 3 * v).long().clamp_(max=v - 1)
    lift = torch.rand((n, 1), generator=gen, device=DEV) * 12.0
    w = weight[target]
    hidden = torch.randn((n, h), generator=gen, device=DEV)
    hidden += w * (lift / w.square().sum(1, keepdim=True))
    out = torch.rand(n, generator=gen, device=DEV) if case["reduction"] == "none" else None
    if case["ignored"]:
        target[torch.rand(n, generator=gen, device=DEV) < case["ignored"]] = IGNORE
    kind = TYPES[case["type"]]
    return hidden.to(kind), weight.to(kind), target, out


class _Layout:
    """Where a case's gradients lie in a flat buffer."""

    def __init__(self, case):
        self.shapes = _shapes(case)
        self.numel = [math.prod(s) for s in self.shapes]
        step = 1 if case.get("packed") else ALIGN
        self.at, self.total = [], 0
        for n in self.numel:
            self.at.append(self.total)
            self.total += -(-n // step) * step

    def views(self, flat):
        return [flat[o:o + n].view(s) for o, n, s in zip(self.at, self.numel, self.shapes)]


def _flat(case, L, seed):
    gen = _generator(seed)
    flat = torch.empty(L.total, dtype=TYPES[case["type"]], device=DEV)
    for a in range(0, L.total, 1 << 28):
        part = flat[a:a + (1 << 28)]
        part.copy_(torch.randn(part.numel(), generator=gen, device=DEV).mul_(case["std"]))
    return flat


def _limit(case, L):
    """About half the gradients' norm: what clipping has to cut."""
    n = sum(L.numel)
    return 0.5 * case["std"] * {1.0: 0.8 * n, 2.0: math.sqrt(n), math.inf: 1.0}[case["norm_type"]]


def prepare(case, seed):
    state = {"call": case["call"]}
    if case["call"] in ("loss", "grad"):
        hidden, weight, target, out = _head(case, seed)
        train = case["call"] == "grad"
        state.update(hidden=hidden.requires_grad_(train), weight=weight.requires_grad_(train),
                     target=target, out=out, reduction=case["reduction"])
        return state
    L = _Layout(case)
    state.update(flat=_flat(case, L, seed), norm_type=case["norm_type"], limit=_limit(case, L))
    state["params"] = [torch.nn.Parameter(torch.empty_like(g)) for g in L.views(state["flat"])]
    for p, g in zip(state["params"], L.views(state["flat"])):
        p.grad = g
    return state


# -- one pass -------------------------------------------------------------------


def run(state):
    call = state["call"]
    if call == "loss":
        return _run_loss(state)
    if call == "grad":
        return _run_grad(state)
    if call == "norm":
        grads = [p.grad for p in state["params"]]
        if own:
            import luma_amd
            return [luma_amd.get_total_norm(grads, state["norm_type"])]
        return [_plain_norm(grads, state["norm_type"])]
    # (a pass over the gradients of the pass before has something to cut again)
    limit, state["limit"] = state["limit"], state["limit"] * 0.999
    if own:
        import luma_amd
        norm = luma_amd.clip_grad_norm_(state["params"], limit, state["norm_type"])
    else:
        grads = [p.grad for p in state["params"]]
        norm = _plain_norm(grads, state["norm_type"])
        part = (limit / (norm + 1e-6)).clamp(max=1.0)
        [g.copy_(g.float() * part) for g in grads]
    return [state["flat"], norm]


def _run_loss(state):
    if own:
        import luma_amd
        return [luma_amd.linear_cross_entropy(state["hidden"], state["weight"], state["target"],
                                              IGNORE, state["reduction"])]
    return [_plain_loss(state)[0]]


def _run_grad(state):
    if own:
        import luma_amd
        loss = luma_amd.linear_cross_entropy(state["hidden"], state["weight"], state["target"],
                                             IGNORE, state["reduction"])
        got = torch.autograd.grad(loss, (state["hidden"], state["weight"]), state["out"])
        return [loss.detach(), *got]
    with torch.no_grad():
        loss, d, x, w = _plain_loss(state, True)
        return [loss, (d @ w).to(state["hidden"].dtype), (d.T @ x).to(state["weight"].dtype)]


def _plain_loss(state, grad=False):
    """The loss from whole float32 logits; with grad, the logits' gradient
    (written over them) and the float32 operands too."""
    x, w, target = state["hidden"].detach().float(), state["weight"].detach().float(), state["target"]
    logits = x @ w.T
    keep = target != IGNORE
    at = torch.where(keep, target, 0)[:, None]
    top = logits.max(1, keepdim=True).values
    picked = logits.gather(1, at)
    e = logits.sub_(top).exp_()
    total = e.sum(1, keepdim=True)
    loss = torch.where(keep, (top + total.log() - picked)[:, 0], 0.0)
    each = torch.ones_like(loss)
    if state["reduction"] == "none":
        each = state["out"] if grad else each
        value = loss
    elif state["reduction"] == "sum":
        value = loss.sum()
    else:
        value = loss.sum() / keep.sum()
        each = each / keep.sum()
    if not grad:
        return (value,)
    d = e.div_(total)
    d.scatter_add_(1, at, torch.full_like(picked, -1.0))
    d.mul_(torch.where(keep, each, 0.0)[:, None])
    return value, d, x, w


def _plain_norm(grads, norm_type):
    if norm_type == math.inf:
        return torch.stack([g.float().abs().amax() for g in grads]).amax()
    if norm_type == 1.0:
        return torch.stack([g.float().abs().sum() for g in grads]).sum()
    return torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()


def work(case):
    """The loss: both operands read once, 2 operations for each of a logit's
    products; its gradient: both gradients written, and their products.  A norm
    reads the gradients, clipping writes them too."""
    size = TYPES[case["type"]].itemsize
    if case["call"] in ("loss", "grad"):
        n, h, v = case["tokens"], case["hidden"], case["vocab"]
        train = case["call"] == "grad"
        return {"bytes": (n * h + v * h) * size * (2 if train else 1) + 12 * n,
                "flops": (6 if train else 2) * n * h * v}
    n = sum(_Layout(case).numel)
    clip = case["call"] == "clip"
    return {"bytes": n * size * (2 if clip else 1), "flops": n * (3 if clip else 2)}


# -- the same in 64 bits --------------------------------------------------------


def exact(case, seed):
    if case["call"] in ("loss", "grad"):
        return _exact_loss(case, seed)
    L = _Layout(case)
    flat = _flat(case, L, seed)
    # (a buffer's padding is not part of any gradient)
    inside = torch.zeros(L.total, dtype=torch.bool, device=DEV)
    for o, n in zip(L.at, L.numel):
        inside[o:o + n] = True
    p, norm = case["norm_type"], 0.0
    for a in range(0, L.total, 1 << 28):
        part = flat[a:a + (1 << 28)][inside[a:a + (1 << 28)]].double()
        if part.numel():
            got = float(torch.linalg.vector_norm(part, p))
            norm = max(norm, got) if p == math.inf else norm + got ** p
    norm = torch.tensor(norm if p == math.inf else norm ** (1.0 / p), dtype=torch.float64,
                        device=DEV)
    if case["call"] == "norm":
        return [norm]
    out = flat.double()
    out[inside] *= min(1.0, _limit(case, L) / (float(norm) + 1e-6))
    return [out, norm]


def _exact_loss(case, seed):
    hidden, weight, target, out = _head(case, seed)
    n, w = case["tokens"], weight.double()
    valid = target != IGNORE
    losses = torch.zeros(n, dtype=torch.float64, device=DEV)
    train = case["call"] == "grad"
    d_w = torch.zeros_like(w) if train else None
    d_x = []
    for a in range(0, n, 1024):
        x, rows = hidden[a:a + 1024].double(), valid[a:a + 1024].nonzero()[:, 0]
        words = target[a:a + 1024][rows]
        logp = torch.log_softmax(x @ w.T, dim=1)
        losses[a + rows] = -logp[rows, words]
        if train:
            share = torch.zeros(len(x), dtype=torch.float64, device=DEV)
            share[rows] = {"none": lambda: out[a + rows].double(),
                           "sum": lambda: torch.ones(len(rows), dtype=torch.float64, device=DEV),
                           "mean": lambda: torch.full((len(rows),), 1.0 / max(1, int(valid.sum())),
                                                      dtype=torch.float64, device=DEV)
                           }[case["reduction"]]()
            p = logp.exp_()
            p[rows, words] -= 1.0
            p *= share[:, None]
            d_x.append(p @ w)
            d_w += p.T @ x
    loss = {"none": lambda: losses, "sum": losses.sum,
            "mean": lambda: losses.sum() / valid.sum()}[case["reduction"]]()
    return [loss, torch.cat(d_x), d_w] if train else [loss]
