"""linear_cross_entropy's 16-bit gradients for gradients of the loss of any
size, against the formulas in 64 bits.

The tolerances are test_gpu_xent's, which scale with the loss's gradient, but
for float16's smallest step: half of it, 2^-25, and 2^-38 of the largest token
gradient in D.  A float16 result is an infinity from 65520 on, half a step
above the largest number; a float32 one below 2^-126 is off by half of 2^-149
more."""

import pytest
import torch

from luma_amd import linear_cross_entropy
from test_gpu_xent import IGNORE, Exact, _inputs, _within

pytestmark = pytest.mark.gpu

LARGEST = 65520.0


def _grads(x, w, t, g, reduction):
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    return torch.autograd.grad(linear_cross_entropy(a, b, t, IGNORE, reduction), (a, b), g)


def _compare(got, ref):
    for name, y, want, tol in (("d_hidden", got[0], ref.d_x, ref.tol_x),
                               ("d_weight", got[1], ref.d_w, ref.tol_w)):
        _within(y, want, tol, name)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [40, 100, 700])       # D in two parts; in one; in larger tiles
@pytest.mark.parametrize("scale", [2.0 ** -8, 1.0, 3.0, 2.0 ** 8])
def test_a_gradient_for_each_token(scale, n, dtype):
    x, w, t = _inputs(n, 64, 300, dtype, seed=31, ignored=0.2)
    gen = torch.Generator(device="cuda").manual_seed(32)
    g = (torch.rand(n, generator=gen, device="cuda") + 0.5) * scale
    _compare(_grads(x, w, t, g, "none"), Exact(x, w, t, g))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [40, 700])
def test_token_gradients_far_apart(n, dtype):
    """From 2^-20 to 1, some negative."""
    x, w, t = _inputs(n, 64, 300, dtype, seed=33)
    gen = torch.Generator(device="cuda").manual_seed(34)
    g = torch.exp2(-20.0 * torch.rand(n, generator=gen, device="cuda"))
    g[::3] *= -1.0
    _compare(_grads(x, w, t, g, "none"), Exact(x, w, t, g))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [40, 100, 700])
@pytest.mark.parametrize("reduction,scale", [("mean", 65536.0), ("mean", 1.0), ("sum", 2.0 ** -8),
                                             ("sum", 2.0 ** 8), ("sum", -3.0)])
def test_one_gradient_for_all_tokens(reduction, scale, n, dtype):
    """GradScaler's factor over a mean, and sums."""
    x, w, t = _inputs(n, 64, 300, dtype, seed=35, ignored=0.2)
    count = int((t != IGNORE).sum()) if reduction == "mean" else 1
    g = torch.full((n,), scale / count, dtype=torch.float64, device="cuda")
    got = _grads(x, w, t, torch.tensor(scale, device="cuda"), reduction)
    ref = Exact(x, w, t, g)
    # (the mean's division is a float32 one)
    ref.tol_x, ref.tol_w = 1.0001 * ref.tol_x, 1.0001 * ref.tol_w
    _compare(got, ref)


@pytest.mark.parametrize("reduction", ["none", "sum"])
@pytest.mark.parametrize("n", [40, 100])
def test_float16_past_its_range(n, reduction):
    """2^-40: every gradient is below half of float16's smallest step; 2^40: infinities
    where the formula's value is past the largest number, the others as they are."""
    x, w, t = _inputs(n, 64, 300, torch.float16, seed=36)
    for scale in (2.0 ** -40, 1e-38):
        g = torch.full((n,), scale, device="cuda")
        ref = Exact(x, w, t, g)
        assert float(ref.d_x.abs().max()) < 2.0 ** -26 > float(ref.d_w.abs().max())
        for y in _grads(x, w, t, g if reduction == "none" else g[0], reduction):
            assert not y.any()
    g = torch.full((n,), 2.0 ** 40, device="cuda")
    got = _grads(x, w, t, g if reduction == "none" else g[0], reduction)
    ref = Exact(x, w, t, g)
    for y, want, tol in ((got[0], ref.d_x, ref.tol_x), (got[1], ref.d_w, ref.tol_w)):
        past = want.abs() - tol >= LARGEST
        assert bool(past.any())
        assert torch.equal(y[past].double(), torch.sign(want[past]) * float("inf"))
        low = want.abs() + tol < LARGEST
        assert bool(((y.double() - want).abs() <= tol)[low].all())
        assert not bool(y.isnan().any())


@pytest.mark.parametrize("n", [40, 100])
def test_float32_among_the_smallest_numbers(n):
    x, w, t = _inputs(n, 64, 300, torch.float32, seed=37)
    gen = torch.Generator(device="cuda").manual_seed(38)
    g = (torch.rand(n, generator=gen, device="cuda") + 0.5) * 1e-38
    assert bool((g > 0).all())
    ref = Exact(x, w, t, g)
    ref.tol_x, ref.tol_w = ref.tol_x + 2.0 ** -149, ref.tol_w + 2.0 ** -149
    _compare(_grads(x, w, t, g, "none"), ref)
