"""layer_norm, add_layer_norm and dropout against their formulas in 64 bits.

Tolerances, from the operations (e = 2^-24; u = half a unit in the last place
of a result's type: 2^-24, 2^-8 for bfloat16, 2^-11 for float16, whose smallest
step adds 2^-25).

* A lane adds the elements of a row that it holds one after the other, at most
  q = 32 of them (8 ceil(h / 8192) past 16,384), the lanes' sums go up a tree of
  six, and at most 16 wavefronts' sums follow each other: a sum of positive terms
  is within (q + 22) e of itself, any sum within (q + 22) e of the terms' sizes.
* So, relative to the deviation, the mean of the differences is within
  (q + 22) e, the deviation within (q + 22) e / 2 + 4 e, an element's difference
  within 2 e |z| + e: z is within ez = (q + 26) e (1 + |z|) (1 + k)^2, where
  k = (q + 22) e |m| r is how far the first mean, about which the differences are
  taken, can be off (in deviations: 1 is reached where a row stands 3e5 of them
  from 0).  The backward reads the mean rounded to float32, which adds e |m| r.
* y = z w + b: |w| ez + 2 e (|z w| + |y|) + u |y|.
* d_s = r (g - mean(g) - z mean(g z)) + d_total: r (4 e (|g| + |mean(g)| +
  |z mean(g z)|) + (q + 23) e mean|g| + |z| (mean(|g| ez) + (q + 23) e mean|g z|)
  + ez |mean(g z)|) + (q + 26) e |r (...)| + 2 e (|d_s| + |d_total|) + u |d_s|.
* d_weight: a register takes a workgroup's rows one after the other, then the
  workgroup's teams and 1 / 32 of the workgroups, then 32: at most t terms in a
  row; sum |d_y| ez + (t + 2) e sum |d_y z| + u |d_weight|; d_bias without the
  first part.
"""

import math

import pytest
import torch
import torch.nn.functional as F

import luma_amd
import residual_util
from luma_amd import _lib as L
from luma_amd import add_layer_norm, dropout, layer_norm

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
DTYPES = list(UNIT)
EPS = 1e-5


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=_gen(seed), device="cuda") * scale).to(dtype)


def _within(got, want, tol, what):
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    off = (got.double() - want).abs()
    worst = float((off / tol.clamp(min=1e-300)).max()) if off.numel() else 0.0
    assert bool((off <= tol).all()), f"{what}: {worst:.3g} times the tolerance"


class Exact:
    """y, and the gradients for d_y and d_total, of the norm of s."""

    def __init__(self, s, w, b, out, d_y=None, d_total=None, eps=EPS):
        n, h = s.shape
        s = s.detach().double()
        wd = torch.ones(h, dtype=torch.float64, device="cuda") if w is None else w.detach().double()
        bd = torch.zeros_like(wd) if b is None else b.detach().double()
        q = 32 if h <= 16384 else 8 * -(-h // 8192)
        m = s.mean(1, keepdim=True)
        r = ((s - m).square().mean(1, keepdim=True) + eps).rsqrt()
        z = (s - m) * r
        ez = (q + 26) * E * (1.0 + z.abs()) * (1.0 + (q + 22) * E * m.abs() * r).square()
        self.y = z * wd + bd
        self.tol_y = (wd.abs() * ez + 2 * E * ((z * wd).abs() + self.y.abs())
                      + UNIT[out] * self.y.abs() + TINY[out])
        if d_y is None:
            return
        ez = ez + E * m.abs() * r
        d = d_y.double()
        g = d * wd
        mg, mgz = g.mean(1, keepdim=True), (g * z).mean(1, keepdim=True)
        self.d_s = r * (g - mg - z * mgz)
        self.tol_s = (r * (4 * E * (g.abs() + mg.abs() + (z * mgz).abs())
                           + (q + 23) * E * g.abs().mean(1, keepdim=True)
                           + z.abs() * ((g.abs() * ez).mean(1, keepdim=True)
                                        + (q + 23) * E * (g * z).abs().mean(1, keepdim=True))
                           + ez * mgz.abs()) + (q + 26) * E * self.d_s.abs())
        if d_total is not None:
            self.d_s = self.d_s + d_total.double()
            self.tol_s = self.tol_s + 2 * E * (self.d_s.abs() + d_total.double().abs())
        self.d_w, self.d_b = (d * z).sum(0), d.sum(0)
        t = n + 64 if n < 1024 else -(-n // 256) + 64
        self.tol_w = (d.abs() * ez).sum(0) + (t + 2) * E * (d * z).abs().sum(0)
        self.tol_b = (t + 2) * E * d.abs().sum(0)


def _check_norm(x, w, b, out, seed=3, eps=EPS):
    d_y = _randn(x.shape, seed, out)
    ref = Exact(x, w, b, out, d_y, eps=eps)
    leaves = [t.clone().requires_grad_() for t in (x, w, b) if t is not None]
    rest = iter(leaves[1:])
    y = layer_norm(leaves[0], None if w is None else next(rest), None if b is None else next(rest),
                   eps, dtype=out)
    assert y.dtype == out and y.is_contiguous()
    _within(y.detach(), ref.y, ref.tol_y, "y")
    got = iter(torch.autograd.grad(y, leaves, d_y))
    u = UNIT[x.dtype]
    d_x = next(got)
    assert d_x.dtype == x.dtype
    _within(d_x, ref.d_s, ref.tol_s + u * ref.d_s.abs() + TINY[x.dtype], "d_x")
    for t, want, tol, name in ((w, "d_w", "tol_w", "d_weight"), (b, "d_b", "tol_b", "d_bias")):
        if t is None:
            continue
        d = next(got)
        assert d.dtype == t.dtype
        want = getattr(ref, want)
        _within(d, want, getattr(ref, tol) + UNIT[t.dtype] * want.abs() + TINY[t.dtype], name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [1, 2, 7, 8, 63, 64, 65, 100, 128, 129, 257, 512, 515, 768, 1001, 1024,
                               2047, 2048, 4096, 4100, 8191, 8192, 8193, 12288, 16384, 16385, 20001])
def test_widths(h, dtype):
    """Every team's narrowest, widest and odd rows, and rows that no team holds."""
    n = 37 if h < 2048 else 5
    _check_norm(_randn((n, h), 1, dtype, 2.0) + 0.5, _randn((h,), 2, dtype) + 1, _randn((h,), 4, dtype),
                dtype)


@pytest.mark.parametrize("n", [1, 2, 3, 31, 33, 255, 256, 257, 4097, 100001])
@pytest.mark.parametrize("h", [3, 24, 300])
def test_rows(n, h):
    _check_norm(_randn((n, h), 1), _randn((h,), 2) + 1, _randn((h,), 4), torch.float32)


@pytest.mark.parametrize("h", [100, 768, 5000, 17000])
@pytest.mark.parametrize("branch", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wide", [False, True])
def test_mixed_types(h, branch, wide):
    """A float32 stream into a 16-bit branch, parameters of either type."""
    param = torch.float32 if wide else branch
    _check_norm(_randn((50, h), 1), _randn((h,), 2, param) + 1, _randn((h,), 4, param), branch)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_without_parameters(weight, bias, dtype):
    w = _randn((200,), 2, dtype) if weight else None
    b = _randn((200,), 4, dtype) if bias else None
    _check_norm(_randn((60, 200), 1, dtype), w, b, dtype)
    _check_norm(_randn((4, 20000), 1, dtype), None, None, dtype)


@pytest.mark.parametrize("mean", [0.0, 1000.0])
@pytest.mark.parametrize("scale", [0.0, 1e-4, 1.0, 1e4])
@pytest.mark.parametrize("h", [96, 4096, 17001])
def test_scales(scale, mean, h):
    """Constant rows, rows far from 0, small and large ones."""
    _check_norm(_randn((40, h), 1, scale=scale) + mean, _randn((h,), 2), _randn((h,), 4),
                torch.float32)
    _check_norm(_randn((40, h), 1, scale=scale) + mean, _randn((h,), 2), _randn((h,), 4),
                torch.float32, eps=1e-12 if scale else 1e-5)


def _drop64(x, res, p, seed, call, out):
    keep = residual_util.kept(x.shape, p, seed, call).cuda()
    part = torch.where(keep, x.double() / (1.0 - p) if p < 1.0 else 0.0, 0.0)
    y = part if res is None else res.double() + part
    return keep, y, 4 * E * part.abs() + E * y.abs() + UNIT[out] * y.abs() + TINY[out]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 1000, 1001, 2048 * 8 + 5, 300001])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(n, dtype, p):
    x, g = _randn((n,), 1, dtype).requires_grad_(), _randn((n,), 2, dtype)
    seed, call = 0x123456789ABCDEF + n, n
    y = dropout(x, p, seed, call)
    keep, want, tol = _drop64(x.detach(), None, p, seed, call, dtype)
    assert y.dtype == dtype and bool((y[~keep] == 0).all())
    _within(y.detach(), want, tol, "y")
    d_x, = torch.autograd.grad(y, x, g)
    _, want, tol = _drop64(g, None, p, seed, call, dtype)
    assert d_x.dtype == dtype and bool((d_x[~keep] == 0).all())
    _within(d_x, want, tol, "d_x")


def test_dropout_large():
    """The kernel that takes four eights a thread, an odd length and the limit's
    low half (p 2^32 is 429496730: its halves are 6553 and 39322)."""
    n = (1 << 21) * 2 + 4099
    x = _randn((n,), 1).requires_grad_()
    for p in (0.1, 3.0 / 65536):
        y = dropout(x, p, -5, 1)
        keep, want, tol = _drop64(x.detach(), None, p, (1 << 64) - 5, 1, torch.float32)
        assert torch.equal(y.detach() != 0, keep & (x.detach() != 0))
        _within(y.detach(), want, tol, "y")
        share = float(keep.double().mean())
        assert abs(share - (1 - p)) < 6 * math.sqrt(p * (1 - p) / n)


def test_the_second_block_decides():
    """Elements whose high half is the limit's: p is set to lie within them."""
    n, seed = 1 << 20, 99
    drawn = residual_util.bits(0, n, seed, 0)
    for at in (5, 77777, n - 1):
        u = int(drawn[at])
        x = torch.ones(n, device="cuda")
        for limit in (u, u + 1):                        # kept, dropped
            p = limit / 2.0 ** 32
            y = dropout(x, p, seed)
            assert bool(y[at] != 0) == (limit == u)
            assert torch.equal((y != 0).cpu(), torch.from_numpy(drawn >= limit))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("n", [5, 4096, 2500007])
def test_dropout_onto_a_residual(n, dtype, wide):
    stream = torch.float32 if wide else dtype
    x, res = _randn((n,), 1, dtype).requires_grad_(), _randn((n,), 2, stream).requires_grad_()
    y = dropout(x, 0.3, 17, 3, residual=res)
    assert y.dtype == stream
    keep, want, tol = _drop64(x.detach(), res.detach(), 0.3, 17, 3, stream)
    _within(y.detach(), want, tol, "y")
    g = _randn((n,), 4, stream)
    d_x, d_res = torch.autograd.grad(y, (x, res), g)
    assert d_x.dtype == dtype and torch.equal(d_res, g)
    _, want, tol = _drop64(g, None, 0.3, 17, 3, dtype)
    _within(d_x, want, tol, "d_x")


def _check_add(n, h, stream, branch, p, param=None, seed=31, call=2):
    param = param or branch
    x, res = _randn((n, h), 1, branch).requires_grad_(), _randn((n, h), 2, stream, 2.0).requires_grad_()
    w, b = (_randn((h,), 3, param) + 1).requires_grad_(), _randn((h,), 4, param).requires_grad_()
    y, total = add_layer_norm(x, res, w, b, EPS, p, seed, call)
    assert y.dtype == branch and total.dtype == stream
    keep, want, tol = _drop64(x.detach(), res.detach(), p, seed, call, stream)
    _within(total.detach(), want, tol, "total")
    d_y, d_total = _randn((n, h), 5, branch), _randn((n, h), 6, stream)
    ref = Exact(total, w, b, branch, d_y, d_total)
    _within(y.detach(), ref.y, ref.tol_y, "y")
    d_x, d_res, d_w, d_b = torch.autograd.grad((y, total), (x, res, w, b), (d_y, d_total))
    _within(d_res, ref.d_s, ref.tol_s + UNIT[stream] * ref.d_s.abs() + TINY[stream], "d_residual")
    scale = keep / (1.0 - p)
    want = ref.d_s * scale
    _within(d_x, want, ref.tol_s * scale + (4 * E + UNIT[branch]) * want.abs() + TINY[branch], "d_x")
    _within(d_w, ref.d_w, ref.tol_w + UNIT[param] * ref.d_w.abs() + TINY[param], "d_weight")
    _within(d_b, ref.d_b, ref.tol_b + UNIT[param] * ref.d_b.abs() + TINY[param], "d_bias")


@pytest.mark.parametrize("stream,branch", [(d, d) for d in DTYPES]
                         + [(torch.float32, torch.bfloat16), (torch.float32, torch.float16)])
@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("n,h", [(1, 1), (3, 7), (100, 96), (33, 129), (9, 768), (17, 1001), (5, 4096),
                                 (3, 9001), (2, 16385)])
def test_add_layer_norm(n, h, p, stream, branch):
    _check_add(n, h, stream, branch, p, torch.float32 if n % 2 else branch)


@pytest.mark.parametrize("n,h", [(8192, 768), (3000, 4099)])
def test_add_layer_norm_of_many_rows(n, h):
    _check_add(n, h, torch.float32, torch.bfloat16, 0.1, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("h", [40, 1003])
def test_one_call_is_the_two(dtype, h):
    """The same mask, the same sum, the same norm, bit for bit, both ways."""
    x, res = _randn((70, h), 1, dtype).requires_grad_(), _randn((70, h), 2, dtype).requires_grad_()
    w, b = _randn((h,), 3).requires_grad_(), _randn((h,), 4).requires_grad_()
    y, total = add_layer_norm(x, res, w, b, EPS, 0.4, 7, 5)
    total2 = dropout(x, 0.4, 7, 5, residual=res)
    y2 = layer_norm(total2, w, b, EPS)
    assert torch.equal(total, total2) and torch.equal(y, y2)
    g = _randn(y.shape, 6, dtype)
    for p, q in zip(torch.autograd.grad(y, (x, res, w, b), g),
                    torch.autograd.grad(y2, (x, res, w, b), g)):
        # (the sum's gradient is rounded once on the way to x in one call, twice in two)
        assert torch.equal(p, q) or dtype != torch.float32
        assert bool(((p.double() - q.double()).abs() <= 2 * UNIT[dtype] * q.double().abs()
                     + TINY[dtype]).all())


@pytest.mark.parametrize("p", [0.0, 0.5])
def test_a_branch_that_is_its_residual(p):
    """Both gradients go to one leaf (without draws they are one tensor)."""
    x = _randn((12, 40), 1).requires_grad_()
    a, b = (x.detach().clone().requires_grad_() for _ in range(2))
    g, t = _randn((12, 40), 2), _randn((12, 40), 3)
    d, = torch.autograd.grad(add_layer_norm(x, x, p=p, seed=1), x, (g, t))
    d_a, d_b = torch.autograd.grad(add_layer_norm(a, b, p=p, seed=1), (a, b), (g, t))
    assert torch.equal(d, d_a + d_b)
    (add_layer_norm(x, x, p=p, seed=1)[0] * g).sum().backward()
    add_layer_norm(a, b, p=p, seed=1)[0].backward(g)
    assert torch.equal(x.grad, a.grad + b.grad)
    if p == 0.0:
        assert a.grad.data_ptr() != b.grad.data_ptr()
    d, = torch.autograd.grad(dropout(x, p, 1, residual=x), x, g)
    d_a, d_b = torch.autograd.grad(dropout(a, p, 1, residual=b), (a, b), g)
    assert torch.equal(d, d_a + d_b)


def test_unused_results():
    x, res = _randn((20, 64), 1).requires_grad_(), _randn((20, 64), 2).requires_grad_()
    w = _randn((64,), 3).requires_grad_()
    y, total = add_layer_norm(x, res, w, p=0.5, seed=3)
    g = _randn((20, 64), 4)
    keep = residual_util.kept((20, 64), 0.5, 3, 0).cuda()
    d_x, d_res, d_w = torch.autograd.grad(total, (x, res, w), g, retain_graph=True)
    assert torch.equal(d_res, g) and torch.equal(d_x, torch.where(keep, g * 2, 0.0))
    assert bool((d_w == 0).all())
    # one of the gradients alone
    whole = torch.autograd.grad(y, (x, res, w), g, retain_graph=True)
    for leaf, want in zip((x, res, w), whole):
        assert torch.equal(torch.autograd.grad(y, leaf, g, retain_graph=True)[0], want)


def test_leading_dimensions_and_strides():
    base = _randn((4, 6, 40, 3), 1)
    for x in (base[..., :40, 0], base.transpose(1, 3)[..., 0], base[:, ::2, :, 1],
              _randn((4, 6, 50), 2)[..., 3:43], _randn((1, 40), 3).expand(9, 40),
              _randn((40,), 4), _randn((6, 40), 5)[::2], _randn((40, 6), 6).T,
              torch._neg_view(_randn((6, 40), 7)), torch._efficientzerotensor((6, 40), device="cuda")):
        w = _randn((x.shape[-1],), 8)
        want = layer_norm(x.clone().contiguous(), w)
        assert torch.equal(layer_norm(x, w), want)
        y, total = add_layer_norm(x, x, w, p=0.2, seed=1)
        c = x.clone().contiguous()
        y2, total2 = add_layer_norm(c, c, w, p=0.2, seed=1)
        assert torch.equal(y, y2) and torch.equal(total, total2)
        assert torch.equal(dropout(x, 0.3, 4, residual=x), dropout(c, 0.3, 4, residual=c))
    x = _randn((6, 80), 9).requires_grad_()
    y = layer_norm(x[:, ::2])
    d, = torch.autograd.grad(y.sum(), x, retain_graph=True)  # an expanded gradient
    d2, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(d, d2) and bool((d[:, 1::2] == 0).all())


@pytest.mark.parametrize("offset", [1, 3, 5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_alignment(offset, dtype):
    """Operands that begin anywhere."""
    h, n = 136, 11
    x = _randn((n * h + 8,), 1, dtype)[offset:offset + n * h].view(n, h)
    w = _randn((h + 8,), 2, dtype)[offset:offset + h]
    assert torch.equal(layer_norm(x, w, w), layer_norm(x.clone(), w.clone(), w.clone()))
    assert torch.equal(dropout(x, 0.5, 1), dropout(x.clone(), 0.5, 1))


def test_empty():
    for shape in ((0, 8), (3, 0, 8)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda", requires_grad=True)
        y = layer_norm(x, w)
        assert y.shape == x.shape
        d_x, d_w = torch.autograd.grad(y.sum(), (x, w))
        assert d_x.shape == x.shape and bool((d_w == 0).all())
        y, total = add_layer_norm(x, x, w, p=0.1)
        assert y.shape == total.shape == x.shape
        assert dropout(x, 0.5, 0).shape == x.shape


def test_not_a_number():
    """A row with an infinity or a NaN is NaN, and no other; dropped elements reach
    nothing."""
    x = _randn((20, 300), 1)
    x[3, 5], x[7, 299], x[11, 0] = math.inf, math.nan, -math.inf
    y = layer_norm(x, _randn((300,), 2))
    bad = torch.tensor([3, 7, 11], device="cuda")
    good = torch.ones(20, dtype=torch.bool, device="cuda")
    good[bad] = False
    assert bool(y[bad].isnan().all()) and bool(y[good].isfinite().all())
    keep = residual_util.kept((20, 300), 0.5, 8, 0).cuda()
    z = torch.where(keep, _randn((20, 300), 3), math.nan)
    assert bool(dropout(z, 0.5, 8).isfinite().all())
    assert bool(add_layer_norm(z, _randn((20, 300), 4), p=0.5, seed=8)[0].isfinite().all())
    assert bool((dropout(torch.full((100,), math.inf, device="cuda"), 1.0, 0) == 0).all())


def test_seeds():
    """A seed on the device, negative and unsigned seeds, calls."""
    x = torch.ones(10000, device="cuda")
    at = torch.tensor(-7, device="cuda")
    assert torch.equal(dropout(x, 0.5, at, 3), dropout(x, 0.5, -7, 3))
    assert torch.equal(dropout(x, 0.5, (1 << 64) - 7, 3), dropout(x, 0.5, -7, 3))
    assert not torch.equal(dropout(x, 0.5, -7, 4), dropout(x, 0.5, -7, 3))
    assert torch.equal(add_layer_norm(x.view(100, 100), x.view(100, 100), p=0.5, seed=at)[1],
                       add_layer_norm(x.view(100, 100), x.view(100, 100), p=0.5, seed=-7)[1])
    y = x.requires_grad_()
    z = dropout(y, 0.5, at)
    at += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()


def test_repeatable():
    x, w = _randn((5000, 777), 1).requires_grad_(), _randn((777,), 2).requires_grad_()
    g = _randn((5000, 777), 3)
    first = torch.autograd.grad(layer_norm(x, w), (x, w), g)
    for _ in range(3):
        for p, q in zip(torch.autograd.grad(layer_norm(x, w), (x, w), g), first):
            assert torch.equal(p, q)


def test_against_differences():
    """Differences of the float32 kernels' outputs along a direction v.  Their
    rounding is at most the sum of |c| tol_y over the step; what a difference of
    this step is off the gradient by, the same difference in 64 bits tells."""
    n, h, step = 6, 50, 2.0 ** -7
    x, w, b = _randn((n, h), 1), _randn((h,), 2) + 1, _randn((h,), 3)
    c = _randn((n, h), 4)
    for which in range(3):
        v = torch.sign(_randn((x, w, b)[which].shape, 5))
        sides, sides64 = [], []
        rounding = 0.0
        for sign in (1.0, -1.0):
            args = [x, w, b]
            args[which] = args[which] + sign * step * v
            sides.append(float((layer_norm(*args).double() * c).sum()))
            ref = Exact(*args, torch.float32)
            sides64.append(float((ref.y * c).sum()))
            rounding += float((ref.tol_y * c.abs()).sum())
        got = (sides[0] - sides[1]) / (2 * step)
        want = (sides64[0] - sides64[1]) / (2 * step)
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        grad = torch.autograd.grad(layer_norm(*leaves), leaves, c)[which]
        ref = Exact(x, w, b, torch.float32, c)
        exact = (ref.d_s, ref.d_w, ref.d_b)[which]
        tol = (ref.tol_s, ref.tol_w, ref.tol_b)[which] + E * exact.abs()
        along = float((grad.double() * v).sum())
        assert abs(got - want) <= rounding / (2 * step)
        assert abs(along - want) <= float(tol.sum()) + abs(float((exact * v).sum()) - want)


def test_differentiated_again():
    x, w = _randn((8, 32), 1).requires_grad_(), _randn((32,), 2).requires_grad_()
    for f, name in ((lambda: layer_norm(x, w), "layer_norm"),
                    (lambda: add_layer_norm(x, x, w, p=0.5)[0], "add_layer_norm"),
                    (lambda: dropout(x, 0.5, 0), "dropout")):
        d, = torch.autograd.grad(f().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match=f"{name}: its gradients cannot"):
            d.sum().backward()


def test_inference_and_no_grad():
    x, w = _randn((8, 32), 1).requires_grad_(), _randn((32,), 2).requires_grad_()
    want = layer_norm(x, w)
    with torch.no_grad():
        got = layer_norm(x, w)
        assert torch.equal(got, want) and not got.requires_grad
    with torch.inference_mode():
        got = layer_norm(x, w)
        assert torch.equal(got, want) and got.is_inference()
        y, total = add_layer_norm(got, got, w, p=0.5, seed=1)
        assert torch.equal(dropout(got, 0.5, 1, residual=got), total)


def test_mutated_operands():
    x, w = _randn((8, 32), 1).requires_grad_(), _randn((32,), 2).requires_grad_()
    y = layer_norm(x, w)
    with torch.no_grad():
        x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_mutated_results():
    """The sum is what the backward reads: a program that writes to it is told so."""
    x, res = _randn((8, 32), 1).requires_grad_(), _randn((8, 32), 2)
    y, total = add_layer_norm(x, res, p=0.5, seed=1)
    total.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    z = dropout(x, 0.5, 1)
    z.mul_(2.0)                                   # (nothing of it is kept)
    keep = residual_util.kept((8, 32), 0.5, 1, 0).cuda()
    d, = torch.autograd.grad(z.sum(), x)
    assert torch.equal(d, keep * 4.0)


def test_another_stream():
    x, w = _randn((3000, 640), 1).requires_grad_(), _randn((640,), 2).requires_grad_()
    g = _randn((3000, 640), 3)
    want_y = layer_norm(x, w)
    want = torch.autograd.grad(want_y, (x, w), g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(10):
            y = layer_norm(x, w)
            got = torch.autograd.grad(y, (x, w), g)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want_y) and all(torch.equal(p, q) for p, q in zip(got, want))


def test_captured_training_step():
    """Forward and backward in one graph, the seed advanced on the device: every
    replay is the eager call of that seed."""
    n, h = 300, 200
    x, res = _randn((n, h), 1).requires_grad_(), _randn((n, h), 2).requires_grad_()
    w, b = _randn((h,), 3).requires_grad_(), _randn((h,), 4).requires_grad_()
    g = _randn((n, h), 5)
    seed = torch.tensor(100, device="cuda")

    def step(seed):
        y, total = add_layer_norm(x, res, w, b, p=0.3, seed=seed, call=1)
        z = dropout(y, 0.2, seed, 2, residual=total)
        return [z.detach(), *torch.autograd.grad(z, (x, res, w, b), g)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(seed)
    torch.cuda.current_stream().wait_stream(s)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(seed)
        seed += 1
    with torch.cuda.graph(other):       # (one that shares its memory's pool and runs between)
        rest = step(5)
    want_rest = [t.clone() for t in step(5)]
    for replay in range(4):
        graph.replay()
        got = [t.clone() for t in out]
        other.replay()
        torch.cuda.synchronize()
        want = step(100 + replay)
        assert all(torch.equal(p, q) for p, q in zip(got, want)), replay
        assert all(torch.equal(p, q) for p, q in zip(rest, want_rest)), replay
        with torch.no_grad():
            x.mul_(1.01)
        want_rest = [t.clone() for t in step(5)]


def test_many_rows():
    """More rows than one launch has threads for, elements past 2^31; the last rows
    are the eager call's on those alone."""
    n, h = (1 << 28) + 37, 8
    x = torch.empty((n, h), dtype=torch.bfloat16, device="cuda")
    x[:1000], x[-1000:] = _randn((1000, h), 1), _randn((1000, h), 2)
    w = _randn((h,), 3, torch.bfloat16)
    y = layer_norm(x, w)
    for part in (slice(0, 1000), slice(n - 1000, n)):
        assert torch.equal(y[part], layer_norm(x[part].clone(), w))
    y = dropout(x, 0.5, 3)
    first = (n - 1000) * h
    keep = residual_util.kept((1000, h), 0.5, 3, 0, first).cuda()
    assert torch.equal(y[-1000:], torch.where(keep, x[-1000:] * 2, 0.0))
    del y
    y, total = add_layer_norm(x, x, w, p=0.5, seed=3)
    want = torch.where(keep, x[-1000:].float() * 2, 0.0) + x[-1000:].float()
    assert torch.equal(total[-1000:], want.bfloat16())
    assert torch.equal(y[-1000:], layer_norm(total[-1000:].clone(), w))


def test_a_block_and_the_loss():
    """The operators as a model runs them: a branch onto the stream, the last norm,
    the head's loss; gradients of everything against float64."""
    n, h, v = 64, 96, 50
    gen = _gen(11)
    embed, mix, head = (torch.randn(s, generator=gen, device="cuda") * 0.3
                        for s in ((n, h), (h, h), (v, h)))
    weights = [torch.randn(h, generator=gen, device="cuda") * 0.1 + 1 for _ in range(2)]
    biases = [torch.randn(h, generator=gen, device="cuda") * 0.1 for _ in range(2)]
    target = torch.randint(0, v, (n,), generator=gen, device="cuda")
    keep = residual_util.kept((n, h), 0.1, 5, 1).cuda()

    def model(own, embed, mix, head, w0, w1, b0, b1):
        if own:
            y = layer_norm(embed, w0, b0)
            y, x = add_layer_norm(y @ mix, embed, w1, b1, p=0.1, seed=5, call=1)
            return luma_amd.linear_cross_entropy(y + x, head, target)
        y = F.layer_norm(embed, (h,), w0, b0)
        x = embed + (y @ mix) * (keep / 0.9)
        return F.cross_entropy((F.layer_norm(x, (h,), w1, b1) + x) @ head.T, target)

    leaves = [t.clone().requires_grad_() for t in (embed, mix, head, *weights, *biases)]
    doubles = [t.double().requires_grad_() for t in leaves]
    loss, want = model(True, *leaves), model(False, *[t for t in doubles])
    assert abs(float(loss) - float(want)) < 1e-5
    for p, q in zip(torch.autograd.grad(loss, leaves), torch.autograd.grad(want, doubles)):
        assert float((p.double() - q).norm() / q.norm()) < 1e-5


def test_without_the_host_module(monkeypatch):
    """The operators' own path gives the same bits."""
    x, res = _randn((40, 100), 1).requires_grad_(), _randn((40, 100), 2).requires_grad_()
    w, b = _randn((100,), 3).requires_grad_(), _randn((100,), 4).requires_grad_()
    g = _randn((40, 100), 5)

    def calls():
        y = layer_norm(x, w, b)
        z, total = add_layer_norm(x, res, w, b, p=0.3, seed=2)
        k, t = add_layer_norm(x, res, w, b)
        d = dropout(x, 0.3, torch.tensor(2, device="cuda"), residual=res)
        out = [y, z, total, k, t, d]
        grads = []
        for o in (y, z, total, k, t, d):
            grads += torch.autograd.grad(o, (x, res, w, b), g, retain_graph=True, allow_unused=True)
        return out + grads

    want = calls()
    monkeypatch.setattr(L, "host_calls", lambda: None)
    for p, q in zip(calls(), want):
        assert (p is None) == (q is None) and (p is None or torch.equal(p, q))
