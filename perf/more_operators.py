"""The operators around a model's residual stream and on its tokens'
log-probabilities, as cases to be timed and compared.

``norm`` is layer normalisation (``luma_amd.layer_norm``), ``drop`` is dropout
whose mask is drawn from a counter-based generator and never stored
(``luma_amd.dropout``), ``add`` is both at the border of two blocks: the
branch's output, dropped out, is added to the residual stream and the sum is
normalised for the next branch (``luma_amd.add_layer_norm``).  ``policy`` is
the clipped policy loss with a KL term on the log-probabilities of sampled
tokens (``luma_amd.policy_loss``).

A case's fields: ``call`` and ``train`` (with the gradients).  For ``norm`` and
``add``: ``rows``, ``width``, ``stream`` and ``branch`` (the residual stream's
type and that of what a branch reads and writes), ``param`` (the type of weight
and bias), ``p``.  For ``drop``: ``rows``, ``width``, ``branch``, ``stream``
(the residual's and the result's type; none without a residual), ``p``.  For
``policy``: ``sequences``, ``length``, ``type``, ``each`` (an advantage for each
token and not for each sequence), ``ref`` (with the KL term), ``ragged`` (a mask
of lengths, some of them 0), ``reduction``.
"""

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-5
LOW, HIGH, KL = 0.2, 0.28, 0.04
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# -- the cases ------------------------------------------------------------------


def _norm(name, rows, width, stream, branch=None, param="float32", train=True):
    return {"name": name, "call": "norm", "train": train, "rows": rows, "width": width,
            "stream": stream, "branch": branch or stream, "param": param, "p": 0.0}


def _add(name, rows, width, stream, branch, p, param="float32", train=True):
    return dict(_norm(name, rows, width, stream, branch, param, train), call="add", p=p)


def _drop(name, rows, width, branch, p, stream=None, train=True):
    return {"name": name, "call": "drop", "train": train, "rows": rows, "width": width,
            "branch": branch, "stream": stream, "p": p}


def _policy(name, sequences, length, reduction, train=True, kind="float32", each=False, ref=True,
            ragged=True):
    return {"name": name, "call": "policy", "train": train, "sequences": sequences,
            "length": length, "type": kind, "each": each, "ref": ref, "ragged": ragged,
            "reduction": reduction}


def listed():
    return [
        # the nanoGPT-sized model's norms (32 windows of 64 tokens): latency
        _norm("norm nano", 2048, 128, "float32"),
        # one token's hidden state of the Llama-3-8B-sized width, in evaluation: latency
        _norm("norm one token", 1, 4096, "bfloat16", param="bfloat16", train=False),
        # odd rows of odd width in half precision, a training step
        _norm("norm ragged fp16", 1021, 1001, "float16", param="float16"),
        # GPT-2 small's blocks under mixed precision: the stream is float32, dropout 0.1
        _add("add gpt2 mixed", 8192, 768, "float32", "bfloat16", 0.1),
        # a wide model's training step in pure bfloat16 without dropout: the largest norm
        _add("add llama bf16", 16384, 4096, "bfloat16", "bfloat16", 0.0, param="bfloat16"),
        # its evaluation over a stream of float32, no gradients
        _add("add llama eval", 8192, 4096, "float32", "bfloat16", 0.0, train=False),
        # GPT-2 small's attention weights, 8 windows of 12 heads: the largest dropout
        _drop("drop attention", 8 * 12 * 1024, 1024, "bfloat16", 0.1),
        # the nanoGPT-sized model's embeddings: latency
        _drop("drop nano", 2048, 128, "float32", 0.2),
        # a branch of odd size onto its residual in half precision, forward only
        _drop("drop residual fp16", 4095, 1001, "float16", 0.3, "float16", train=False),
        # a small batch of answers, an advantage for each: latency
        _policy("policy small", 16, 65, "mean"),
        # a large batch of long answers, each counting the same, with ragged lengths
        _policy("policy large", 512, 8192, "sequence"),
        # the loss of each token, with each token's advantage, for a log: no gradients
        _policy("policy log", 61, 4097, "none", train=False, each=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges."""
    call = rng.choice(["norm", "add", "drop", "policy"])
    train = rng.random() < 0.7
    if call == "policy":
        b, t = _log_uniform(rng, 1, 512), _log_uniform(rng, 1, 8192)
        return {"call": call, "train": train, "sequences": b, "length": t,
                "type": rng.choice(["float32", "float32", "bfloat16", "float16"]),
                "each": rng.random() < 0.5, "ref": rng.random() < 0.7,
                "ragged": rng.random() < 0.7,
                "reduction": rng.choice(["mean", "sequence", "sum", "none"])}
    branch = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    stream = rng.choice(["float32", branch])
    rows, width = _log_uniform(rng, 1, 100000), _log_uniform(rng, 1, 16384)
    if rng.random() < 0.5:
        width = max(8, width // 8 * 8)
    while rows * width > 1 << 26:
        rows = (rows + 1) // 2
    p = rng.choice([0.0, 0.1, rng.uniform(0.0, 0.6)])
    if call == "drop":
        return {"call": call, "train": train, "rows": rows, "width": width, "branch": branch,
                "stream": rng.choice([None, stream]), "p": p}
    return {"call": call, "train": train, "rows": rows, "width": width, "stream": stream,
            "branch": branch, "param": rng.choice(["float32", branch]),
            "p": p if call == "add" else 0.0}


# -- inputs ---------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _stream(gen, rows, width):
    """A residual stream: each token's size is its own, a few channels are far
    larger than the others, and the mean is not 0."""
    x = torch.randn((rows, width), generator=gen, device=DEV)
    x *= torch.rand((rows, 1), generator=gen, device=DEV) * 3.0 + 0.5
    large = torch.rand(width, generator=gen, device=DEV) < 0.004
    x *= torch.where(large, 20.0, 1.0)
    return x.add_(torch.randn(width, generator=gen, device=DEV) * 0.5)


def _stream_inputs(case, seed):
    gen = _generator(seed)
    n, h = case["rows"], case["width"]
    branch = TYPES[case["branch"]]
    stream = TYPES[case["stream"]] if case["stream"] else None
    s = {"p": case["p"], "seed": int(seed) * 0x9E3779B97F4A7C15 % (1 << 63),
         "layer": int(seed) % 61}
    if case["call"] == "norm":
        s["x"] = _stream(gen, n, h).to(stream)
    else:
        s["x"] = torch.randn((n, h), generator=gen, device=DEV).to(branch)
        s["residual"] = _stream(gen, n, h).to(stream) if stream else None
    if case["call"] != "drop":
        param = TYPES[case["param"]]
        s["weight"] = (torch.randn(h, generator=gen, device=DEV) * 0.1 + 1.0).to(param)
        s["bias"] = (torch.randn(h, generator=gen, device=DEV) * 0.1).to(param)
    if case["train"]:
        # (the gradient of a mean over tokens, as GradScaler or the head's scale leaves it)
        grad = torch.randn((n, h), generator=gen, device=DEV) * 0.01
        s["d_y"] = grad.to(stream or branch if case["call"] == "drop" else branch)
        if case["call"] == "add":
            s["d_total"] = (torch.randn((n, h), generator=gen, device=DEV) * 0.01).to(stream)
    return s


def _policy_inputs(case, seed):
    """Log-probabilities of sampled tokens under three policies that lie near each
    other; what stands behind an answer's end is whatever the batch was filled with."""
    gen = _generator(seed)
    b, t = case["sequences"], case["length"]
    kind = TYPES[case["type"]]
    lp = torch.rand((b, t), generator=gen, device=DEV).add_(1e-4).log_()
    old = lp + torch.randn((b, t), generator=gen, device=DEV) * 0.15
    ref = lp + torch.randn((b, t), generator=gen, device=DEV) * 0.3 if case["ref"] else None
    advantage = torch.randn((b, t) if case["each"] else (b,), generator=gen, device=DEV)
    mask = None
    if case["ragged"]:
        length = torch.rand((b, 1), generator=gen, device=DEV) * (t + 1)
        length *= torch.rand((b, 1), generator=gen, device=DEV) >= 0.05
        length[0].clamp_(min=1.0)      # (a batch without any token has no mean)
        mask = torch.arange(t, device=DEV)[None] < length.floor()
        old[~mask] = -math.inf
    out = torch.rand((b, t), generator=gen, device=DEV) if case["reduction"] == "none" else None
    return {"logp": lp.to(kind), "old": old.to(kind), "ref": None if ref is None else ref.to(kind),
            "advantage": advantage, "mask": mask, "out": out}


def prepare(case, seed):
    s = _policy_inputs(case, seed) if case["call"] == "policy" else _stream_inputs(case, seed)
    s.update(call=case["call"], train=case["train"], branch=TYPES[case.get("branch", "float32")],
             reduction=case.get("reduction"))
    s["leaves"] = [s[k] for k in ("x", "residual", "weight", "bias", "logp")
                   if s.get(k) is not None]
    if case["train"]:
        for leaf in s["leaves"]:
            leaf.requires_grad_()
    return s


# -- one pass -------------------------------------------------------------------


def run(state):
    call = state["call"]
    if own:
        return _own(state)
    with torch.no_grad():
        if call == "drop":
            return _plain_drop(state)
        if call == "policy":
            return _plain_policy(state)
        return _plain_norm(state)


def _own(s):
    import luma_amd
    call = s["call"]
    if call == "policy":
        loss = luma_amd.policy_loss(s["logp"], s["old"], s["advantage"], s["mask"], s["ref"],
                                    clip_low=LOW, clip_high=HIGH, kl_weight=KL,
                                    reduction=s["reduction"])
        if not s["train"]:
            return [loss]
        return [loss.detach(), *torch.autograd.grad(loss, s["leaves"], s["out"])]
    if call == "norm":
        out = [luma_amd.layer_norm(s["x"], s["weight"], s["bias"], EPS, dtype=s["branch"])]
        grads = ["d_y"]
    elif call == "drop":
        out = [luma_amd.dropout(s["x"], s["p"], s["seed"], s["layer"], residual=s["residual"])]
        grads = ["d_y"]
    else:
        out = list(luma_amd.add_layer_norm(s["x"], s["residual"], s["weight"], s["bias"], EPS,
                                           p=s["p"], seed=s["seed"], call=s["layer"]))
        grads = ["d_y", "d_total"]
    if not s["train"]:
        return out
    return [*(y.detach() for y in out),
            *torch.autograd.grad(out, s["leaves"], [s[g] for g in grads])]


M0, M1, W0, W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
MASK = 0xFFFFFFFF


def _philox(block, stream, layer, seed):
    """The eight 16-bit halves of each Philox4x32-10 block, [blocks, 8]."""
    c = [block & MASK, block >> 32, torch.full_like(block, stream), torch.full_like(block, layer)]
    k0, k1 = seed & MASK, seed >> 32 & MASK
    for _ in range(10):
        # (the 64-bit products wrap; their halves are right all the same)
        p0, p1 = c[0] * M0, c[2] * M1
        c = [(p1 >> 32 & MASK) ^ c[1] ^ k0, p1 & MASK, (p0 >> 32 & MASK) ^ c[3] ^ k1, p0 & MASK]
        k0, k1 = k0 + W0 & MASK, k1 + W1 & MASK
    return torch.stack([w >> s & 0xFFFF for w in c for s in (0, 16)], dim=1)


def _plain_kept(shape, p, seed, layer):
    """Which elements are kept: the element's 32 bits are not below p 2^32."""
    n = math.prod(shape)
    block = torch.arange((n + 7) // 8, device=DEV)
    bits = (_philox(block, 0, layer, seed) << 16) + _philox(block, 1, layer, seed)
    return (bits >= int(math.floor(p * 2.0 ** 32 + 0.5))).view(-1)[:n].view(shape)


def _plain_drop(s):
    x, p = s["x"].float(), s["p"]
    kept = _plain_kept(x.shape, p, s["seed"], s["layer"])
    y = torch.where(kept, x * (1.0 / (1.0 - p)), 0.0)
    if s["residual"] is not None:
        y = s["residual"].float() + y
    out = [y.to(s["x"].dtype if s["residual"] is None else s["residual"].dtype)]
    if s["train"]:
        out.append(torch.where(kept, s["d_y"].float() * (1.0 / (1.0 - p)), 0.0).to(s["x"].dtype))
        if s["residual"] is not None:
            out.append(s["d_y"].clone())
    return out


def _plain_norm(s):
    x, w = s["x"], s["weight"].float()
    out, kept, scale = [], None, 1.0 / (1.0 - s["p"])
    if s["call"] == "add":
        y = x.float()
        if s["p"]:
            kept = _plain_kept(x.shape, s["p"], s["seed"], s["layer"])
            y = torch.where(kept, y * scale, 0.0)
        # (the sum is an output of its own; its norm is that of the sum as it is kept)
        x = (s["residual"].float() + y).to(s["residual"].dtype)
        out = [x]
    x = x.float()
    h = x.shape[1]
    centred = x - x.sum(1, keepdim=True) / h
    r = ((centred * centred).sum(1, keepdim=True) / h + EPS).rsqrt()
    xh = centred * r
    out.insert(0, (xh * w + s["bias"].float()).to(s["branch"]))
    if not s["train"]:
        return out
    d = s["d_y"].float()
    g = d * w
    dx = r * (g - g.sum(1, keepdim=True) / h - xh * ((g * xh).sum(1, keepdim=True) / h))
    if s["call"] == "add":
        dx = dx + s["d_total"].float()
        part = dx if kept is None else torch.where(kept, dx * scale, 0.0)
        out.append(part.to(s["x"].dtype))
        out.append(dx.to(s["residual"].dtype))
    else:
        out.append(dx.to(s["x"].dtype))
    out.append((d * xh).sum(0).to(s["weight"].dtype))
    out.append(d.sum(0).to(s["bias"].dtype))
    return out


def _plain_policy(s):
    a = s["advantage"] if s["advantage"].dim() == 2 else s["advantage"][:, None]
    lp, mask = s["logp"].float(), s["mask"]
    # (64 bits: a ratio at its limit falls to one side or the other)
    d = s["logp"].double() - s["old"].double()
    if mask is not None:
        d = torch.where(mask, d, 0.0)
    up, low = d > math.log1p(HIGH), d < math.log1p(-LOW)
    r = d.float().exp()
    cut = torch.where(up, 1.0 + HIGH, torch.where(low, 1.0 - LOW, r))
    held = torch.where(a > 0, up, low & (a < 0))
    value = -torch.where(held, cut, r) * a
    grad = torch.where(held, 0.0, -r * a)
    if s["ref"] is not None:
        q = s["ref"].float() - lp
        e = torch.expm1(q)
        value = value + KL * (e - q)
        grad = grad - KL * e
    if mask is not None:
        value = torch.where(mask, value, 0.0)
        grad = torch.where(mask, grad, 0.0)
    share = torch.ones_like(lp) if mask is None else mask.float()
    if s["reduction"] == "none":
        out = value
        share = share if s["out"] is None else s["out"]
    else:
        if s["reduction"] == "mean":
            share = share / share.sum()
        elif s["reduction"] == "sequence":
            count = share.sum(1, keepdim=True)
            share = share / count.clamp(min=1.0) / (count > 0).sum()
        out = (value * share).sum()
    return [out, (grad * share).to(s["logp"].dtype)] if s["train"] else [out]


def work(case):
    """Every input read once, every output written once; the operations are those
    on an element in 32 bits (the generator's are whole numbers)."""
    if case["call"] == "policy":
        n, size = case["sequences"] * case["length"], TYPES[case["type"]].itemsize
        token = size * (3 if case["ref"] else 2) + (1 if case["ragged"] else 0)
        token += 4 if case["each"] else 0
        if case["reduction"] == "none":
            token += 4 + (4 if case["train"] else 0)
        if case["train"]:
            token += size
        return {"bytes": n * token + 4 * case["sequences"],
                "flops": n * (25 if case["train"] else 15)}
    n, branch = case["rows"] * case["width"], TYPES[case["branch"]].itemsize
    stream = TYPES[case["stream"]].itemsize if case["stream"] else 0
    if case["call"] == "drop":
        one = branch + (2 * stream if stream else branch)
        # (a residual's gradient is the result's own)
        if case["train"]:
            one += (stream or branch) + branch
        return {"bytes": n * one, "flops": n * (4 if case["train"] else 2)}
    one = stream + branch
    if case["call"] == "add":
        one += stream + branch
    if case["train"]:
        # d_y and the stream's gradient; with a branch also d_total and the branch's gradient
        one += branch + stream
        if case["call"] == "add":
            one += stream + (branch if case["p"] or case["branch"] != case["stream"] else 0)
    small = 2 * case["width"] * TYPES[case["param"]].itemsize
    return {"bytes": n * one + small * (2 if case["train"] else 1),
            "flops": n * (22 if case["train"] else 8)}


# -- the same in 64 bits --------------------------------------------------------


def _exact_kept(shape, p, seed, layer):
    """The same draws, with 16-bit limbs and a block's words one after the other."""
    n = math.prod(shape)
    kept = torch.empty(((n + 7) // 8, 8), dtype=torch.bool, device=DEV)
    limit = round(p * 2 ** 32)

    def wide(a, m):
        low, high = (a & 65535) * m, (a >> 16) * m
        mid = (low >> 16) + (high & 0xFFFFFFFFFFFF)
        return mid >> 16, (mid & 65535) << 16 | low & 65535

    for a in range(0, len(kept), 1 << 22):
        index = torch.arange(a, min(len(kept), a + (1 << 22)), device=DEV)
        words = []
        for stream in range(2):
            x0, x1 = index % (1 << 32), index // (1 << 32)
            x2, x3 = torch.zeros_like(index) + stream, torch.zeros_like(index) + layer
            for i in range(10):
                h0, l0 = wide(x0, M0)
                h1, l1 = wide(x2, M1)
                x0 = h1 ^ x1 ^ ((seed % (1 << 32)) + i * W0) % (1 << 32)
                x2 = h0 ^ x3 ^ ((seed >> 32) + i * W1) % (1 << 32)
                x1, x3 = l1, l0
            words.append((x0, x1, x2, x3))
        for i, (top, below) in enumerate(zip(*words)):
            for j in range(2):
                u = (top >> 16 * j) % 65536 * 65536 + (below >> 16 * j) % 65536
                kept[a:a + len(index), 2 * i + j] = ~(u < limit)
    return kept.reshape(-1)[:n].reshape(shape)


def exact(case, seed):
    if case["call"] == "policy":
        return _exact_policy(case, _policy_inputs(case, seed))
    s = _stream_inputs(case, seed)
    names = [k for k in ("x", "residual", "weight", "bias") if s.get(k) is not None]
    leaf = {k: s[k].double().requires_grad_(case["train"]) for k in names}
    x, out = leaf["x"], []
    if case["call"] != "norm":
        if s["p"]:
            x = x * (_exact_kept(x.shape, s["p"], s["seed"], s["layer"]) / (1.0 - s["p"]))
        if "residual" in leaf:
            x = leaf["residual"] + x
        out = [x]
    if case["call"] != "drop":
        if case["call"] == "add":
            x = x + (x.detach().to(s["residual"].dtype).double() - x.detach())
        out.insert(0, torch.nn.functional.layer_norm(x, x.shape[1:], leaf["weight"], leaf["bias"],
                                                     EPS))
    if not case["train"]:
        return [y.detach() for y in out]
    grads = [s[k].double() for k in ("d_y", "d_total") if k in s]
    got = torch.autograd.grad(out, [leaf[k] for k in names], grads)
    return [*(y.detach() for y in out), *got]


def _exact_policy(case, s):
    lp = s["logp"].double().requires_grad_()
    rows = torch.arange(lp.numel(), device=DEV).view(lp.shape)
    mask = torch.ones_like(lp, dtype=torch.bool) if s["mask"] is None else s["mask"]
    at = rows[mask]
    a = s["advantage"].double()
    a = (a if a.dim() == 2 else a[:, None].expand(lp.shape)).reshape(-1)[at]
    here = lp.reshape(-1)[at]
    ratio = (here - s["old"].double().reshape(-1)[at]).exp()
    each = -a * ratio
    each = torch.where((a >= 0) & (ratio > 1.0 + HIGH), -a * (1.0 + HIGH), each)
    each = torch.where((a < 0) & (ratio < 1.0 - LOW), -a * (1.0 - LOW), each)
    if s["ref"] is not None:
        q = s["ref"].double().reshape(-1)[at] - here
        each = each + KL * (torch.expm1(q) - q)
    if case["reduction"] == "none":
        loss = torch.zeros(lp.numel(), dtype=torch.float64, device=DEV)
        loss = loss.index_copy(0, at, each).view(lp.shape)
    elif case["reduction"] == "sequence":
        owner = at // lp.shape[1]
        count = torch.bincount(owner, minlength=len(lp))
        sums = torch.zeros(len(lp), dtype=torch.float64, device=DEV).index_add(0, owner, each)
        loss = (sums[count > 0] / count[count > 0]).mean()
    else:
        loss = each.sum() if case["reduction"] == "sum" else each.mean()
    if not case["train"]:
        return [loss.detach()]
    return [loss.detach(), *torch.autograd.grad(loss, lp, s["out"])]
