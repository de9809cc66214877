"""linear_cross_entropy against its formulas in 64 bits.

Tolerances, from the operations (u = half a unit in the last place of the
operands' type: 2^-24, 2^-8 for bfloat16, 2^-11 for float16).

* A logit is a float32 sum of h products: its error is taken as eight standard
  deviations of a random walk of roundings, dl = 8 sqrt(h) 2^-24 sum_k |x_k w_k|.
* exp, log and the scaling by log2(e) add a few units of 2^-24 of the logits'
  size: 2^-21 (1 + max |l|).  So a loss is within 2 max dl + 2^-21 (1 + max |l|)
  = e, a probability within a factor 1 + 2 e.
* D = g (p - [target]) is rounded to the operands' type: |dD| <= |g| p 2 e +
  u |D|, and float16's smallest steps, 2^-24, are 2^-38 of the largest |g|.
* Each gradient is a float32 sum of products of D, rounded once:
  |dD| |W| + 8 sqrt(terms) 2^-24 |D| |W| + u |gradient| (+ float16's 2^-25).
"""

import math

import pytest
import torch

import luma_amd
from luma_amd import linear_cross_entropy

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = list(UNIT)
IGNORE = -100


def _inputs(n, h, v, dtype, seed=0, ignored=0.0, std=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, h), generator=g, device="cuda")
    w = torch.randn((v, h), generator=g, device="cuda") * (std or 2.0 / math.sqrt(h))
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    if ignored:
        t[torch.rand(n, generator=g, device="cuda") < ignored] = IGNORE
    return x.to(dtype), w.to(dtype), t


class Exact:
    """Loss per token, gradients for token gradients g, and their tolerances."""

    def __init__(self, x, w, t, g=None):
        dtype, (n, h), v = x.dtype, x.shape, w.shape[0]
        u = UNIT[dtype]
        x, w = x.detach().double(), w.detach().double()
        valid = t != IGNORE
        logits = x @ w.T
        lse = torch.logsumexp(logits, 1)
        at = torch.where(valid, t, 0)[:, None]
        self.loss = torch.where(valid, lse - logits.gather(1, at)[:, 0], 0.0)
        dl = 8.0 * math.sqrt(h) * 2.0 ** -24 * (x.abs() @ w.abs().T).amax(1)
        self.tol = 2.0 * dl + 2.0 ** -21 * (1.0 + logits.abs().amax(1))
        if g is None:
            return
        g = torch.where(valid, g.double(), 0.0)[:, None]
        p = (logits - lse[:, None]).exp_()
        d = p.clone()
        d.scatter_add_(1, at, torch.full((n, 1), -1.0, dtype=torch.float64, device="cuda"))
        d *= g
        off = g.abs() * p * (2.0 * self.tol[:, None]) + u * d.abs()
        if dtype == torch.float16:
            off += 2.0 ** -38 * g.abs().amax() * valid[:, None]
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
        self.d_x = d @ w
        self.d_w = d.T @ x
        dd = d.abs()
        self.tol_x = (off @ w.abs() + 8.0 * math.sqrt(v) * 2.0 ** -24 * (dd @ w.abs())
                      + u * self.d_x.abs() + tiny)
        self.tol_w = (off.T @ x.abs() + 8.0 * math.sqrt(n) * 2.0 ** -24 * (dd.T @ x.abs())
                      + u * self.d_w.abs() + tiny)


def _within(got, want, tol, what):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    worst = float((off / tol.clamp(min=1e-300)).max()) if off.numel() else 0.0
    assert bool((off <= tol).all()), f"{what}: {worst:.3g} times the tolerance"


def _check(x, w, t, seed=1):
    """Every reduction's loss, and the gradients of each."""
    n = x.shape[0]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = torch.randn(n, generator=gen, device="cuda")
    count = int((t != IGNORE).sum())
    each = Exact(x, w, t, g)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(a, b, t, IGNORE, "none")
    assert loss.dtype == torch.float32 and loss.shape == t.shape
    _within(loss.detach(), each.loss, each.tol, "loss")
    d_x, d_w = torch.autograd.grad(loss, (a, b), g)
    assert d_x.dtype == x.dtype and d_w.dtype == w.dtype
    _within(d_x, each.d_x, each.tol_x, "d_hidden")
    _within(d_w, each.d_w, each.tol_w, "d_weight")
    total, tol = each.loss.sum(), each.tol.sum() + 2.0 ** -23 * each.loss.sum().abs()
    got = linear_cross_entropy(x, w, t, IGNORE, "sum")
    assert got.dim() == 0
    _within(got, total, tol, "sum")
    mean = linear_cross_entropy(a, b, t, IGNORE)
    if count == 0:
        assert math.isnan(float(mean))
        return
    _within(mean.detach(), total / count, tol / count, "mean")
    m = Exact(x, w, t, torch.full((n,), 0.5 / count, dtype=torch.float64, device="cuda"))
    d_x, d_w = torch.autograd.grad(mean * 0.5, (a, b))
    _within(d_x, m.d_x, m.tol_x * 1.0001, "d_hidden of the mean")
    _within(d_w, m.d_w, m.tol_w * 1.0001, "d_weight of the mean")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h,v", [
    (1, 64, 28), (1, 4096, 1000), (2, 8, 1), (3, 1, 5), (1, 1, 1), (16, 64, 300), (17, 100, 257),
    (64, 128, 28), (65, 72, 513), (128, 256, 1000), (300, 1000, 777), (257, 768, 2100),
    (1000, 40, 33), (33, 65, 129), (129, 7, 255), (640, 136, 4097)])
def test_sizes(n, h, v, dtype):
    _check(*_inputs(n, h, v, dtype, seed=n + h + v))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h,v", [(2048, 72, 6200),      # 256 x 256 tiles of logits
                                   (3100, 4000, 300),     # ... of d_hidden
                                   (70, 4096, 3201),      # ... of d_weight
                                   (12, 520, 20000)])     # few tokens, a split vocabulary
def test_large_tiles(n, h, v, dtype):
    _check(*_inputs(n, h, v, dtype, seed=3))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h,v", [(400, 1100, 500),      # 64 tokens to a workgroup
                                   (200, 3000, 60),       # 16
                                   (40, 2056, 90), (1, 1500, 33), (9, 8191, 31)])
@pytest.mark.parametrize("ignored", [0.0, 0.4])
def test_few_words_and_long_hidden_states(n, h, v, dtype, ignored):
    x, w, t = _inputs(n, h, v, dtype, seed=n, ignored=ignored)
    t[0] = v - 1
    _check(x, w, t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 8, 9, 32, 33, 64, 65])
def test_two_parts_of_few_tokens(n, dtype):
    """Up to 64 tokens a gradient is off by its own rounding alone: half a unit of
    each entry, and the float32 terms' (D's second part holds what the first's
    rounding left, so that u^2 of an entry of D, 2 at most, is lost)."""
    x, w, t = _inputs(n, 72, 900, dtype, seed=n)
    g = torch.rand(n, device="cuda") + 0.5
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    got = torch.autograd.grad(linear_cross_entropy(a, b, t, IGNORE, "none"), (a, b), g)
    ref = Exact(x, w, t, g)
    f32 = Exact(x.float(), w.float(), t, g)
    u = UNIT[dtype]
    for y, want, tol in ((got[0], ref.d_x, f32.tol_x), (got[1], ref.d_w, f32.tol_w)):
        rel = float((y.double() - want).norm() / want.norm())
        assert rel <= (u if n <= 64 else 2.0 * u)
        if n <= 64:
            dd = 2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -22
            slack = dd * (g.max().double() * 2.0) * (w if y is got[0] else x).double().abs().sum(0)
            _within(y, want, 1.01 * u * want.abs() + tol + slack + 2.0 ** -25, "a gradient")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pieces_of_the_vocabulary(dtype):
    """More words than two pieces hold (1 GiB of D each)."""
    n = 8200
    v = 2 * (1 << 30) // (n * (4 if dtype == torch.float32 else 2)) + 777
    _check(*_inputs(n, 40, v, dtype, seed=4))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("share", [0.3, 0.97, 1.0])
def test_ignored_targets(dtype, share):
    x, w, t = _inputs(200, 96, 500, dtype, seed=5, ignored=share)
    if share < 1.0:
        t[7] = 3
    _check(x, w, t)


def test_ignored_tokens_may_hold_anything():
    x, w, t = _inputs(100, 64, 300, torch.bfloat16, seed=6)
    t[10:20] = IGNORE
    want = linear_cross_entropy(x, w, t, IGNORE, "none")
    y = x.clone()
    y[10:15], y[15:20] = math.nan, math.inf
    a, b = y.requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(a, b, t, IGNORE)
    assert torch.equal(linear_cross_entropy(a, b, t, IGNORE, "none"), want)
    d_x, _ = torch.autograd.grad(loss, (a, b))
    assert not d_x[10:20].any() and bool(d_x.isfinite().all())


@pytest.mark.parametrize("bad", [-1, 300, -101, 2 ** 40, -2 ** 63])
def test_targets_outside_the_vocabulary(bad):
    """NaN for that token, nothing read for it, the others as they were."""
    x, w, t = _inputs(100, 64, 300, torch.float32, seed=7)
    want = linear_cross_entropy(x, w, t, IGNORE, "none")
    t[42] = bad
    a = x.clone().requires_grad_()
    got = linear_cross_entropy(a, w, t, IGNORE, "none")
    assert math.isnan(float(got[42]))
    keep = torch.arange(100, device="cuda") != 42
    assert torch.equal(got[keep], want[keep])
    d_x, = torch.autograd.grad(got.sum(), a)
    assert bool(d_x[42].isnan().all()) and bool(d_x[keep].isfinite().all())
    assert math.isnan(float(linear_cross_entropy(x, w, t, IGNORE)))


def test_another_ignore_index():
    x, w, t = _inputs(50, 64, 30, torch.float32, seed=8)
    t[::3] = 5
    got = linear_cross_entropy(x, w, t, 5, "none")
    assert not got[::3].any()
    want = linear_cross_entropy(x, w, t, IGNORE, "none")
    keep = t != 5
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", DTYPES)
def test_logits_of_every_size(dtype):
    """Large logits (the running maximum), -inf ones, and whole rows without
    any finite one."""
    x, w, t = _inputs(40, 64, 700, dtype, seed=9, std=2.0)
    _check(x, w, t)
    x = torch.ones((3, 8), dtype=dtype, device="cuda")
    w = torch.zeros((600, 8), dtype=dtype, device="cuda")
    w[:, 0] = torch.linspace(-4, 4, 600, device="cuda").to(dtype)
    w[5:300, 1] = -math.inf
    t = torch.tensor([2, 400, 7], device="cuda")
    got = linear_cross_entropy(x, w, t, IGNORE, "none")
    keep = torch.cat([w[:5, 0], w[300:, 0]]).double()
    lse = torch.logsumexp(keep, 0)
    for i in (0, 1):
        want = float(lse - w[t[i], 0].double())
        assert abs(float(got[i]) - want) <= 2.0 ** -19
    assert float(got[2]) == math.inf
    w[:, 1] = -math.inf
    assert bool(linear_cross_entropy(x, w, t, IGNORE, "none").isnan().all())
    w[:, 1] = 0.0
    w[9, 1] = math.inf
    assert bool(linear_cross_entropy(x, w, t, IGNORE, "none").isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_not_a_number_stays_in_its_token(dtype):
    x, w, t = _inputs(70, 64, 300, dtype, seed=10)
    want = linear_cross_entropy(x, w, t, IGNORE, "none")
    x[33, 5] = math.nan
    got = linear_cross_entropy(x, w, t, IGNORE, "none")
    keep = torch.arange(70, device="cuda") != 33
    assert math.isnan(float(got[33])) and torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -40, 2.0 ** 40, 1e-38, 0.0])
def test_gradients_of_any_size(scale):
    """float16 keeps D's digits whatever the loss's gradient (GradScaler's
    factor, a mean over many tokens)."""
    x, w, t = _inputs(100, 64, 300, torch.float16, seed=11)
    g = torch.rand(100, device="cuda") + 0.5
    ref = Exact(x, w, t, g)
    a, b = x.float().requires_grad_(), w.float().requires_grad_()
    h, k = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(h, k, t, IGNORE, "none")
    d_x, d_w = torch.autograd.grad(loss, (h, k), g * scale)
    if scale == 1.0:
        _within(d_x, ref.d_x, ref.tol_x, "d_hidden")
    elif scale == 0.0:
        assert not d_x.any() and not d_w.any()
    # in float32 the gradients are those of scale 1 times the scale
    loss = linear_cross_entropy(a, b, t, IGNORE, "none")
    one = torch.autograd.grad(loss, (a, b), g, retain_graph=True)
    got = torch.autograd.grad(loss, (a, b), g * scale)
    if scale in (2.0 ** -40, 2.0 ** 40):
        assert all(torch.equal(o * scale, s) for o, s in zip(one, got))


def test_infinite_gradient_of_one_token():
    x, w, t = _inputs(70, 64, 300, torch.float32, seed=12)
    a = x.clone().requires_grad_()
    g = torch.ones(70, device="cuda")
    want, = torch.autograd.grad(linear_cross_entropy(a, w, t, IGNORE, "none"), a, g)
    g[20] = math.inf
    got, = torch.autograd.grad(linear_cross_entropy(a, w, t, IGNORE, "none"), a, g)
    keep = torch.arange(70, device="cuda") != 20
    assert torch.equal(got[keep], want[keep]) and not bool(got[20].isfinite().any())


def test_against_differences():
    """The gradient along random directions against central differences of the
    loss.  A step of 2^-6 in a direction that changes no logit by more than 1
    per unit: the difference is off by its third derivative, at most
    2^-12 / 6 * 2 per token, and by the two losses' errors over 2^-5."""
    n, h, v = 64, 48, 200
    x, w, t = _inputs(n, h, v, torch.float32, seed=13)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    grads = torch.autograd.grad(linear_cross_entropy(a, b, t, IGNORE, "sum"), (a, b))
    e = 2.0 ** -6
    for seed in range(4):
        g = torch.Generator(device="cuda").manual_seed(100 + seed)
        for k in range(2):
            v_ = torch.randn((x, w)[k].shape, generator=g, device="cuda")
            v_ /= (v_ @ w.T if k == 0 else x @ v_.T).abs().max()
            ends = []
            for sign in (e, -e):
                y, z = (x + sign * v_, w) if k == 0 else (x, w + sign * v_)
                ends.append((float(linear_cross_entropy(y, z, t, IGNORE, "sum")),
                             float(Exact(y, z, t).tol.sum())))
            got = (ends[0][0] - ends[1][0]) / (2 * e)
            want = float((grads[k].double() * v_.double()).sum())
            tol = n * 2.0 ** -12 / 3 + (ends[0][1] + ends[1][1]) / (2 * e) + 1e-5 * abs(want)
            assert abs(got - want) <= tol, (k, got, want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    """Hidden states of all but a sequence's last position, a weight with
    longer rows, operands off every 16-byte boundary: the same results."""
    n, h, v = 90, 72, 333
    x, w, t = _inputs(n, h, v, dtype, seed=14)
    want = linear_cross_entropy(x, w, t, IGNORE, "none")
    big = torch.full((v, h + 5), math.nan, dtype=dtype, device="cuda")
    big[:, 3:3 + h] = w
    flat = torch.full((n * h + 9,), math.nan, dtype=dtype, device="cuda")
    for off in (1, 3, 8):
        flat[off:off + n * h] = x.reshape(-1)
        got = linear_cross_entropy(flat[off:off + n * h].view(n, h), big[:, 3:3 + h], t, IGNORE,
                                   "none")
        assert torch.equal(got, want)
    turned = w.t().contiguous().t()
    assert torch.equal(linear_cross_entropy(x, turned, t, IGNORE, "none"), want)
    seq = torch.full((9, 11, h), math.nan, dtype=dtype, device="cuda")
    seq[:, :-1] = x.view(9, 10, h)
    a = seq.clone().requires_grad_()
    loss = linear_cross_entropy(a[:, :-1], w, t.view(9, 10), IGNORE, "none")
    assert torch.equal(loss.detach(), want.view(9, 10))
    d, = torch.autograd.grad(loss.sum(), a)
    b = x.clone().requires_grad_()
    e, = torch.autograd.grad(linear_cross_entropy(b, w, t, IGNORE, "sum"), b)
    assert torch.equal(d[:, :-1].reshape(n, h), e) and not d[:, -1].any()
    one = linear_cross_entropy(x[:1].expand(5, h), w, t[:1].expand(5), IGNORE, "none")
    assert torch.equal(one, want[:1].expand(5))


def test_only_one_gradient():
    x, w, t = _inputs(100, 64, 300, torch.bfloat16, seed=15)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(linear_cross_entropy(a, b, t), (a, b))
    only_x, = torch.autograd.grad(linear_cross_entropy(a, w, t), a)
    only_w, = torch.autograd.grad(linear_cross_entropy(x, b, t), b)
    assert torch.equal(both[0], only_x) and torch.equal(both[1], only_w)


def test_no_tokens():
    w = torch.randn((30, 16), device="cuda").requires_grad_()
    x = torch.empty((0, 16), device="cuda").requires_grad_()
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    assert math.isnan(float(linear_cross_entropy(x, w, t)))
    assert linear_cross_entropy(x, w, t, IGNORE, "none").shape == (0,)
    loss = linear_cross_entropy(x, w, t, IGNORE, "sum")
    assert float(loss) == 0.0
    d_x, d_w = torch.autograd.grad(loss, (x, w))
    assert d_x.shape == (0, 16) and not d_w.any()


def test_one_token_without_a_batch():
    x, w, t = _inputs(1, 64, 300, torch.float32, seed=16)
    got = linear_cross_entropy(x[0], w, t[0], IGNORE, "none")
    assert got.dim() == 0
    assert torch.equal(got, linear_cross_entropy(x, w, t, IGNORE, "none")[0])


def test_autocast():
    """Under autocast float32 parameters go in as its type and get float32
    gradients."""
    x, w, t = _inputs(100, 64, 300, torch.float32, seed=17)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = linear_cross_entropy(a, b, t)
    loss.backward()
    c, d = x.bfloat16().requires_grad_(), w.bfloat16().requires_grad_()
    want = linear_cross_entropy(c, d, t)
    want.backward()
    assert torch.equal(loss, want)
    assert a.grad.dtype == torch.float32 and torch.equal(a.grad, c.grad.float())
    assert torch.equal(b.grad, d.grad.float())


def test_same_bits_every_time():
    x, w, t = _inputs(700, 200, 5000, torch.bfloat16, seed=18)
    seen = []
    for _ in range(3):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = linear_cross_entropy(a, b, t)
        seen.append((loss.detach(), *torch.autograd.grad(loss, (a, b))))
    for other in seen[1:]:
        assert all(torch.equal(p, q) for p, q in zip(seen[0], other))


def test_graph_and_other_stream():
    x, w, t = _inputs(200, 64, 1000, torch.bfloat16, seed=19)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()

    def step():
        loss = linear_cross_entropy(a, b, t)
        return (loss, *torch.autograd.grad(loss, (a, b)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        y, _, s = _inputs(200, 64, 1000, torch.bfloat16, seed=50 + seed)
        with torch.no_grad():
            a.copy_(y)
        t.copy_(s)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_compile():
    x, w, t = _inputs(100, 64, 300, torch.float32, seed=20)

    def f(x, w, t):
        return linear_cross_entropy(x * 2.0, w, t)

    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = torch.compile(f, fullgraph=True)(a, b, t)
    got = torch.autograd.grad(loss, (a, b))
    want_loss = f(a, b, t)
    want = torch.autograd.grad(want_loss, (a, b))
    assert torch.equal(loss, want_loss)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_without_grad_and_in_inference_mode():
    x, w, t = _inputs(50, 64, 300, torch.bfloat16, seed=22)
    want = linear_cross_entropy(x, w, t)
    with torch.no_grad():
        got = linear_cross_entropy(x.requires_grad_(), w, t)
    assert torch.equal(got, want) and not got.requires_grad
    with torch.inference_mode():
        assert torch.equal(linear_cross_entropy(x.clone(), w.clone(), t.clone()), want)


def test_torch_func_is_refused():
    """torch.func's transforms do not trace the ops (torch.autograd does)."""
    x, w, t = _inputs(50, 64, 300, torch.float32, seed=23)
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda w: linear_cross_entropy(x, w, t))(w)


def test_without_the_host_module(monkeypatch):
    """The custom ops give what the eager path gives."""
    x, w, t = _inputs(100, 64, 300, torch.bfloat16, seed=24)
    outs = []
    for _ in range(2):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = linear_cross_entropy(a, b, t)
        outs.append((loss.detach(), *torch.autograd.grad(loss, (a, b))))
        monkeypatch.setattr(luma_amd._lib, "host_calls", lambda: None)
    assert all(torch.equal(p, q) for p, q in zip(*outs))


@pytest.mark.parametrize("module", [True, False])
def test_gradients_are_not_differentiated_again(module, monkeypatch):
    """create_graph=True gives the same gradients; to differentiate them raises."""
    if not module:
        monkeypatch.setattr(luma_amd._lib, "host_calls", lambda: None)
    x, w, t = _inputs(50, 64, 300, torch.float32, seed=26)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    want = torch.autograd.grad(linear_cross_entropy(a, b, t), (a, b))
    for operands in ((a, b), (a, w), (x, b)):
        loss = linear_cross_entropy(*operands, t)
        leaves = [p for p in operands if p.requires_grad]
        got = torch.autograd.grad(loss, leaves, create_graph=True)
        for p, leaf in zip(got, leaves):
            assert torch.equal(p, want[0] if leaf is a else want[1])
            with pytest.raises(RuntimeError):
                torch.autograd.grad((p ** 2).sum(), leaves, retain_graph=True)


def test_operand_changed_before_the_backward_is_noticed():
    x, w, t = _inputs(50, 64, 300, torch.float32, seed=25)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(a, b, t)
    with torch.no_grad():
        b.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refusals():
    x, w, t = _inputs(10, 16, 30, torch.float32)
    cases = [((x, w, t), dict(reduction="max"), ValueError, "reduction"),
             ((x[:, :8], w, t), {}, ValueError, "do not match"),
             ((x, w, t[:5]), {}, ValueError, "target"),
             ((x, w, t.int()), {}, ValueError, "int64"),
             ((x.double(), w.double(), t), {}, ValueError, "dtype"),
             ((x, w.half(), t), {}, ValueError, "weight"),
             ((x, w[:0], t), {}, ValueError, "empty"),
             ((x.cpu(), w, t), {}, RuntimeError, "ROCm GPU"),
             ((x, w.cpu(), t), {}, RuntimeError, "ROCm GPU"),
             ((x, w, t.cpu()), {}, RuntimeError, "ROCm GPU")]
    for args, more, error, text in cases:
        with pytest.raises(error, match=text):
            linear_cross_entropy(*args, **more)


def test_training_with_the_optimizer():
    """Loss, clipping and step together: a head that learns its targets."""
    x, w, t = _inputs(256, 64, 50, torch.float32, seed=21)
    p = torch.nn.Parameter(w * 0.1)
    opt = luma_amd.LUMA([p], lr=0.05, weight_decay=0.0)
    first = None
    for _ in range(60):
        loss = linear_cross_entropy(x, p, t)
        opt.zero_grad()
        loss.backward()
        luma_amd.clip_grad_norm_([p], 1.0)
        opt.step()
        first = float(loss) if first is None else first
    assert float(loss) < 0.5 * first
