"""policy_loss against its formulas in 64 bits.

Tolerances, from the operations (e = 2^-24; u = half a unit in the last place of
a result's type).  l - l_old is exact in float64 and rounded once, exp within
one unit: r within r (e |d| + 4 e).  q is within e |q|, which moves exp(q) - 1 - q
by e |q| |exp(q) - 1|; the excess itself is within 16 e of itself from its series
(|q| < 1/2), elsewhere within 8 e (exp(q) + 1 + |q|), and exp(q) - 1 within that
and e |q| exp(q).  Products and sums of two add 2 e of each part.  Sums over
tokens are float64; a mean's share is rounded to float32, as the loss is.
"""

import math

import pytest
import torch

import luma_amd
from luma_amd import _lib as L
from luma_amd import linear_cross_entropy, policy_loss

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
REDUCTIONS = ["mean", "sequence", "sum", "none"]
LOW, HIGH, KL = 0.2, 0.3, 0.05


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(shape, seed=0, dtype=torch.float32, each=False, ref=True, ragged=True, spread=0.3):
    g = _gen(seed)
    lp = torch.rand(shape, generator=g, device="cuda").add_(1e-3).log_()
    old = lp + torch.randn(shape, generator=g, device="cuda") * spread
    r = lp + torch.randn(shape, generator=g, device="cuda") * spread if ref else None
    a = torch.randn(shape if each else shape[:-1], generator=g, device="cuda")
    mask = None
    if ragged:
        length = (torch.rand(shape[:-1] + (1,), generator=g, device="cuda") * (shape[-1] + 1)).floor()
        mask = torch.arange(shape[-1], device="cuda") < length
        mask = mask & (torch.rand(shape, generator=g, device="cuda") < 0.9)
    return (lp.to(dtype), old.to(dtype), a, mask, None if r is None else r.to(dtype))


def _within(got, want, tol, what):
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    off = (got.double() - want).abs()
    both = want.isnan() & got.isnan()
    off, tol = torch.where(both, 0.0, off), torch.where(both, 0.0, tol)
    worst = float((off / tol.clamp(min=1e-300)).max()) if off.numel() else 0.0
    assert bool((off <= tol).all()), f"{what}: {worst:.3g} times the tolerance"


class Exact:
    """Values and gradients of the tokens, the loss, its gradient for `out`."""

    def __init__(self, lp, old, a, mask, ref, reduction, out=None, low=LOW, high=HIGH, kl=KL):
        keep = torch.ones_like(lp, dtype=torch.bool) if mask is None else mask
        dtype = lp.dtype
        zero = torch.zeros((), dtype=torch.float64, device="cuda")

        def at(t):
            return torch.where(keep, t.detach().double(), zero)

        lp, old = at(lp), at(old)
        a = a.double() if a.dim() == lp.dim() else a.double()[..., None].expand(lp.shape)
        a = torch.where(keep, a, zero)
        d = lp - old
        r = d.exp()
        clipped = r.clamp(1.0 - low, 1.0 + high)
        value = -torch.minimum(r * a, clipped * a)
        held = torch.minimum(r * a, clipped * a) < r * a
        grad = torch.where(held, zero, -r * a)
        r_off = r * (E * d.abs() + 4 * E)
        v_off = a.abs() * torch.where(held, 2 * E * clipped, r_off + 2 * E * r)
        g_off = torch.where(held, zero, a.abs() * (r_off + 2 * E * r))
        k = moved = zero.expand(lp.shape)

        def excess(x):
            big = x.abs() >= 0.5
            s = torch.expm1(x) - x
            series = x * x * sum(x ** i / math.factorial(i + 2) for i in range(14))
            return big, torch.where(big, s, series)

        big, moved = excess(d)
        moved_off = (E * d.abs() * torch.expm1(d).abs()
                     + torch.where(big, 8 * E * (r + 1 + d.abs()), 16 * E * moved))
        if ref is not None:
            q = at(ref) - lp
            big, k = excess(q)
            k_off = (E * q.abs() * torch.expm1(q).abs()
                     + torch.where(big, 8 * E * (q.exp() + 1 + q.abs()), 16 * E * k))
            value = value + kl * k
            grad = grad - kl * torch.expm1(q)
            v_off = v_off + kl * (k_off + 2 * E * k)
            g_off = g_off + kl * (k_off + E * q.abs() * q.exp() + 4 * E * torch.expm1(q).abs())
            self.kl_off = k_off.sum()
        v_off, g_off = v_off + 2 * E * value.abs(), g_off + 2 * E * grad.abs()
        value, grad = torch.where(keep, value, zero), torch.where(keep, grad, zero)
        v_off, g_off = torch.where(keep, v_off, zero), torch.where(keep, g_off, zero)
        n = keep.sum().double()
        if reduction == "none":
            share = keep.double() if out is None else torch.where(keep, out.double(), zero)
            self.loss, self.tol = value, v_off + E * value.abs()
        else:
            share = keep.double()
            if reduction == "mean":
                share = share / n
            if reduction == "sequence":
                count = keep.sum(-1, keepdim=True).double()
                share = share / count.clamp(min=1.0) / (count > 0).sum()
            self.loss = (value * share).sum()
            self.tol = (v_off * share).sum() + E * self.loss.abs() + 1e-12 * (value * share).abs().sum()
            share = share * (1.0 if out is None else float(out))
        self.grad = torch.where(keep, grad * share, zero)
        self.tol_grad = (g_off * share.abs() + 6 * E * self.grad.abs()
                         + UNIT[dtype] * self.grad.abs() + TINY[dtype])
        self.stats = torch.stack([(held & keep).sum() / n, torch.where(keep, k, zero).sum() / n,
                                  torch.where(keep, moved, zero).sum() / n, n])
        self.tol_stats = torch.stack([E * self.stats[0].abs(),
                                      (self.kl_off if ref is not None else zero) / n,
                                      torch.where(keep, moved_off, zero).sum() / n, zero])
        self.tol_stats = self.tol_stats + 2 * E * self.stats.abs()


def _check(inputs, reduction, **limits):
    lp, old, a, mask, ref = inputs
    leaf = lp.clone().requires_grad_()
    kw = dict(clip_low=LOW, clip_high=HIGH, kl_weight=KL)
    kw.update({{"low": "clip_low", "high": "clip_high", "kl": "kl_weight"}[k]: v
               for k, v in limits.items()})
    loss, stats = policy_loss(leaf, old, a, mask, ref, reduction=reduction, return_stats=True, **kw)
    out = torch.randn(loss.shape, generator=_gen(9), device="cuda")
    want = Exact(lp, old, a, mask, ref, reduction, out, **limits)
    assert loss.dtype == torch.float32 and stats.shape == (4,) and not stats.requires_grad
    _within(loss.detach(), want.loss, want.tol, f"loss ({reduction})")
    _within(stats, want.stats, want.tol_stats, f"stats ({reduction})")
    d, = torch.autograd.grad(loss, leaf, out)
    assert d.dtype == lp.dtype and d.shape == lp.shape
    if not bool(want.loss.isnan().any()):
        _within(d, want.grad, want.tol_grad, f"gradient ({reduction})")
    if mask is not None:
        assert bool((d[~mask] == 0).all())


@pytest.mark.parametrize("reduction", REDUCTIONS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 2), (3, 3), (2, 64), (5, 65), (32, 1024), (33, 7),
                                   (31, 1025), (1, 1024), (1, 5000), (64, 255), (300, 257), (7, 4097),
                                   (9000, 5), (2, 100003), (1, 3000001), (70, 2049), (2100, 1030)])
def test_shapes(shape, reduction):
    """One launch, short rows, pieces of long rows; odd lengths everywhere."""
    _check(_inputs(shape, sum(shape)), reduction)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("each,ref,ragged", [(False, False, False), (True, True, True),
                                             (True, False, True), (False, True, False)])
@pytest.mark.parametrize("shape", [(12, 130), (50, 1500), (3, 4, 90)])
def test_operands(shape, each, ref, ragged, dtype):
    inputs = _inputs(shape, 3, dtype, each, ref, ragged)
    for reduction in REDUCTIONS:
        _check(inputs, reduction)


@pytest.mark.parametrize("reduction", REDUCTIONS)
def test_one_dimension(reduction):
    lp, old, _, mask, ref = _inputs((1, 700), 4)
    a = torch.randn((), generator=_gen(1), device="cuda")
    _check((lp[0], old[0], a, mask[0], ref[0]), reduction)


@pytest.mark.parametrize("reduction", REDUCTIONS)
@pytest.mark.parametrize("limits", [dict(low=0.0, high=0.0), dict(low=1.0, high=5.0),
                                    dict(low=0.5, high=math.inf), dict(kl=0.0), dict(kl=3.0)])
def test_limits(limits, reduction):
    _check(_inputs((20, 200), 5, spread=1.0), reduction, **limits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_the_same_policy(dtype):
    """Ratios of 1 (an update's first pass): nothing is clipped, the divergences are 0."""
    lp, _, a, mask, _ = _inputs((20, 333), 6, dtype)
    leaf = lp.requires_grad_()
    loss, stats = policy_loss(leaf, lp, a, mask, lp, kl_weight=0.1, clip_low=0.0, clip_high=0.0,
                              return_stats=True)
    n = float(mask.sum())
    assert [float(v) for v in stats] == [0.0, 0.0, 0.0, n]
    d, = torch.autograd.grad(loss, leaf)
    want = torch.where(mask, -a[:, None].double() / n, 0.0)
    assert bool(((d.double() - want).abs() <= (4 * E + UNIT[dtype]) * want.abs() + TINY[dtype]).all())


def test_small_divergences_keep_their_digits():
    lp = torch.full((4, 100), -1.0, device="cuda")
    ref = lp + 2.0 ** -12
    a = torch.zeros(4, device="cuda")
    loss, stats = policy_loss(lp, ref, a, None, ref, kl_weight=1.0, return_stats=True)
    q = 2.0 ** -12
    want = q * q / 2 * (1 + q / 3 + q * q / 12)
    assert abs(float(loss) / want - 1) < 16 * E
    assert abs(float(stats[1]) / want - 1) < 16 * E


def test_a_ratio_at_its_limit():
    """The limit's neighbours on both sides, decided in float64."""
    up = math.log1p(0.25)
    near = torch.tensor(up, dtype=torch.float64).float().item()
    steps = [torch.nextafter(torch.tensor(near), torch.tensor(s)).item() for s in (0.0, 1.0)] + [near]
    lp = torch.tensor([steps], device="cuda").requires_grad_()
    loss = policy_loss(lp, torch.zeros_like(lp), torch.ones(1, device="cuda"), clip_high=0.25,
                       reduction="sum")
    d, = torch.autograd.grad(loss, lp)
    for got, x in zip(d[0].tolist(), steps):
        assert (got == 0.0) == (x > up)


def test_masked_places_hold_anything():
    lp, old, a, mask, ref = _inputs((40, 500), 7, each=True)
    mask[5], mask[39] = False, False                  # rows without a token
    want = {}
    for junk in (0.0, math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min):
        args = [torch.where(mask, t, junk) for t in (lp, old, a, ref)]
        leaf = args[0].requires_grad_()
        for reduction in REDUCTIONS:
            loss, stats = policy_loss(leaf, args[1], args[2], mask, args[3], kl_weight=0.1,
                                      reduction=reduction, return_stats=True)
            d, = torch.autograd.grad(loss.sum(), leaf)
            assert bool((d[~mask] == 0).all()) and bool(loss.isfinite().all())
            got = [loss.detach(), stats, d]
            for p, q in zip(got, want.setdefault(reduction, got)):
                assert torch.equal(p, q)


def test_nothing_counts():
    lp, old, a, mask, ref = _inputs((40, 50), 8)
    leaf = lp.requires_grad_()
    for mask in (torch.zeros_like(mask), torch.zeros((40, 1), dtype=torch.bool,
                                                     device="cuda").expand(40, 50)):
        for reduction in REDUCTIONS:
            loss, stats = policy_loss(leaf, old, a, mask, ref, reduction=reduction, return_stats=True)
            d, = torch.autograd.grad(loss.sum(), leaf)
            assert bool((d == 0).all()) and float(stats[3]) == 0
            if reduction in ("mean", "sequence"):
                assert math.isnan(float(loss))
            else:
                assert bool((loss == 0).all())


@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0,)])
def test_empty(shape):
    lp = torch.empty(shape, device="cuda", requires_grad=True)
    a = torch.empty(shape, device="cuda")
    for reduction in REDUCTIONS:
        loss = policy_loss(lp, lp, a, reduction=reduction)
        d, = torch.autograd.grad(loss.sum(), lp)
        assert d.shape == lp.shape
        assert loss.shape == (lp.shape if reduction == "none" else ())


def test_strides_and_alignment():
    """A batch's answers cut out of longer rows, one row for all, one advantage for all."""
    base = [t for t in _inputs((12, 900), 9, each=True)]
    for cut in (slice(1, 900), slice(3, 800), slice(0, 900, 2)):
        args = [t[:, cut] for t in base]
        flat = [t.contiguous() for t in args]
        for reduction in REDUCTIONS:
            got = policy_loss(*args, kl_weight=KL, reduction=reduction)
            assert torch.equal(got, policy_loss(*flat, kl_weight=KL, reduction=reduction))
    lp, old, a, mask, ref = base
    row = old[:1].expand(12, 900)
    assert torch.equal(policy_loss(lp, row, a, mask, ref),
                       policy_loss(lp, row.contiguous(), a, mask, ref))
    one = torch.tensor(0.5, device="cuda")
    assert torch.equal(policy_loss(lp, old, one.expand(12)), policy_loss(lp, old, one.repeat(12)))
    assert torch.equal(policy_loss(lp, old, one.expand(12, 900)),
                       policy_loss(lp, old, one.repeat(12, 900)))
    assert torch.equal(policy_loss(lp, old, a, mask[:, :1].expand(12, 900)),
                       policy_loss(lp, old, a, mask[:, :1].repeat(1, 900)))
    assert torch.equal(policy_loss(lp.T, old.T, a.T, mask.T, ref.T, reduction="sum"),
                       policy_loss(lp.T.contiguous(), old.T.contiguous(), a.T.contiguous(),
                                   mask.T.contiguous(), ref.T.contiguous(), reduction="sum"))


def test_constants():
    """No gradient goes to what the ratios are taken against."""
    lp, old, a, mask, ref = _inputs((6, 40), 10)
    leaves = [t.clone().requires_grad_() for t in (lp, old, a, ref)]
    loss = policy_loss(leaves[0], leaves[1], leaves[2], mask, leaves[3], kl_weight=KL)
    grads = torch.autograd.grad(loss, leaves, allow_unused=True)
    assert grads[0] is not None and all(g is None for g in grads[1:])
    assert not policy_loss(lp, leaves[1], leaves[2], mask, leaves[3]).requires_grad


def test_against_differences():
    """As the norm's: the rounding over the step, and the same difference in 64 bits."""
    lp, old, a, mask, ref = _inputs((5, 60), 11, each=True)
    v = torch.sign(torch.randn(lp.shape, generator=_gen(1), device="cuda"))
    step = 2.0 ** -8
    for reduction in ("mean", "sequence", "sum"):
        sides = []
        for sign in (1.0, -1.0):
            x = lp + sign * step * v
            sides.append((float(policy_loss(x, old, a, mask, ref, clip_low=LOW, clip_high=HIGH,
                                            kl_weight=KL, reduction=reduction)),
                          Exact(x, old, a, mask, ref, reduction)))
        got = (sides[0][0] - sides[1][0]) / (2 * step)
        want = float(sides[0][1].loss - sides[1][1].loss) / (2 * step)
        assert abs(got - want) <= float(sides[0][1].tol + sides[1][1].tol) / (2 * step)
        leaf = lp.clone().requires_grad_()
        d, = torch.autograd.grad(policy_loss(leaf, old, a, mask, ref, clip_low=LOW, clip_high=HIGH,
                                             kl_weight=KL, reduction=reduction), leaf)
        ref64 = Exact(lp, old, a, mask, ref, reduction)
        exact = float((ref64.grad * v).sum())
        along = float((d.double() * v).sum())
        assert abs(along - want) <= float(ref64.tol_grad.sum()) + abs(exact - want)


def test_repeatable():
    inputs = _inputs((600, 2000), 12)
    for reduction in REDUCTIONS:
        first = policy_loss(*inputs, reduction=reduction)
        for _ in range(3):
            assert torch.equal(policy_loss(*inputs, reduction=reduction), first)


def test_differentiated_again():
    lp, old, a, mask, ref = _inputs((6, 40), 13)
    lp.requires_grad_()
    d, = torch.autograd.grad(policy_loss(lp, old, a, mask, ref), lp, create_graph=True)
    with pytest.raises(RuntimeError, match="policy_loss: its gradients cannot"):
        d.sum().backward()


def test_another_stream_and_inference():
    inputs = _inputs((600, 2000), 14)
    want = policy_loss(*inputs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.inference_mode():
        got = policy_loss(*inputs)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize("shape", [(16, 65), (40, 3000)])
def test_captured(shape):
    lp, old, a, mask, ref = _inputs(shape, 15)
    leaf = lp.clone().requires_grad_()

    def step(reduction):
        loss, stats = policy_loss(leaf, old, a, mask, ref, kl_weight=KL, reduction=reduction,
                                  return_stats=True)
        return [loss.detach(), stats, *torch.autograd.grad(loss, leaf)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step("sequence")
    torch.cuda.current_stream().wait_stream(s)
    graphs = {r: torch.cuda.CUDAGraph() for r in ("mean", "sequence")}
    outs = {}
    for reduction, graph in graphs.items():
        with torch.cuda.graph(graph):
            outs[reduction] = step(reduction)
    for replay in range(4):
        for graph in graphs.values():
            graph.replay()
        got = {r: [t.clone() for t in o] for r, o in outs.items()}
        torch.cuda.synchronize()
        for reduction in graphs:
            assert all(torch.equal(p, q) for p, q in zip(got[reduction], step(reduction))), replay
        with torch.no_grad():
            leaf.mul_(1.01)


def test_on_a_heads_log_probabilities():
    """A step as it is used: the head's loss per token, the policy loss on it, and
    the gradients of hidden states and weight, against float64."""
    g = _gen(16)
    b, t, h, v = 6, 50, 64, 200
    x = torch.randn((b, t, h), generator=g, device="cuda")
    w = torch.randn((v, h), generator=g, device="cuda") * 0.2
    words = torch.randint(0, v, (b, t), generator=g, device="cuda")
    a = torch.randn(b, generator=g, device="cuda")
    mask = torch.arange(t, device="cuda") < torch.tensor([50, 3, 0, 21, 49, 1], device="cuda")[:, None]
    with torch.no_grad():
        base = -linear_cross_entropy(x, w, words, reduction="none")
        old = base + torch.randn((b, t), generator=g, device="cuda") * 0.2
        ref = base + torch.randn((b, t), generator=g, device="cuda") * 0.2
    for reduction in ("mean", "sequence"):
        leaves = [s.clone().requires_grad_() for s in (x, w)]
        logp = -linear_cross_entropy(leaves[0], leaves[1], words, reduction="none")
        loss = policy_loss(logp, old, a, mask, ref, clip_low=LOW, clip_high=HIGH, kl_weight=KL,
                           reduction=reduction)
        doubles = [s.double().requires_grad_() for s in (x, w)]
        exact = torch.log_softmax(doubles[0] @ doubles[1].T, -1).gather(-1, words[..., None])[..., 0]
        d = exact.detach() - old.double()
        up = (a[:, None] > 0) & (d > math.log1p(HIGH))
        low = (a[:, None] < 0) & (d < math.log1p(-LOW))
        r = (exact - old.double()).exp()
        value = -torch.where(up, 1 + HIGH, torch.where(low, 1 - LOW, r)) * a[:, None].double()
        q = ref.double() - exact
        value = value + KL * (q.exp() - 1 - q)
        if reduction == "mean":
            want = value[mask].mean()
        else:
            want = torch.stack([value[i][mask[i]].mean() for i in range(b) if mask[i].any()]).mean()
        assert abs(float(loss) - float(want)) < 1e-5 * (1 + abs(float(want)))
        for p, s in zip(torch.autograd.grad(loss, leaves), torch.autograd.grad(want, doubles)):
            assert float((p.double() - s).norm() / s.norm()) < 1e-5


def test_without_the_host_module(monkeypatch):
    inputs = _inputs((40, 1300), 17)
    leaf = inputs[0].clone().requires_grad_()

    def calls():
        got = []
        for reduction in REDUCTIONS:
            loss, stats = policy_loss(leaf, *inputs[1:], kl_weight=KL, reduction=reduction,
                                      return_stats=True)
            got += [loss.detach(), stats, *torch.autograd.grad(loss.sum(), leaf)]
        return got

    want = calls()
    monkeypatch.setattr(L, "host_calls", lambda: None)
    assert all(torch.equal(p, q) for p, q in zip(calls(), want))


def test_public_name():
    assert luma_amd.policy_loss is policy_loss
