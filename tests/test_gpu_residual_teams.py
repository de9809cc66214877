"""The residual stream's operators by the kernel that a width and a size lead to:
one width for each team of lanes that can hold a row, of whole and of cut runs,
with rows for several turns of each team, and operands past the last-level
cache, which have kernels of their own.  Formulas in 64 bits and tolerances are
those of test_gpu_residual.py.
"""

import pytest
import torch

import residual_util
from luma_amd import add_layer_norm, dropout, layer_norm
from test_gpu_residual import EPS, TINY, UNIT, E, Exact, _drop64, _randn, _within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
KINDS = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)]
# Runs of 16 bytes of the stream's type that a row of each team has at most.
RUNS = {F32: [8, 16, 32, 64, 128, 192, 256, 384, 512, 768, 1024, 1536, 2048, 4096],
        BF16: [8, 16, 32, 64, 128, 192, 256, 512, 768, 1024, 1536, 2048]}
RUNS[F16] = RUNS[BF16]


def _widths():
    for stream, branch in KINDS:
        v, last = 16 // stream.itemsize, 0
        for most in RUNS[stream]:
            runs = (last + most + 1) // 2 | 1
            # (the third: rows of float32 that begin where a draw's eight does)
            for h in (runs * v, runs * v - 3) + ((runs * v + 4,) if v == 4 else ()):
                yield pytest.param(stream, branch, h, id=f"{stream}-{branch}-{h}".replace("torch.", ""))
            last = most


def _check(n, h, stream, branch, p, alone=False, seed=77, call=9):
    """add_layer_norm, or (alone) layer_norm of the stream, both ways."""
    res = _randn((n, h), 2, stream, 2.0).add_(0.25).requires_grad_()
    w, b = (_randn((h,), 3, F32) + 1).requires_grad_(), _randn((h,), 4, F32).requires_grad_()
    d_y = _randn((n, h), 5, branch)
    if alone:
        y = layer_norm(res, w, b, EPS, dtype=branch)
        ref = Exact(res, w, b, branch, d_y)
        d_res, d_w, d_b = torch.autograd.grad(y, (res, w, b), d_y)
    else:
        x, d_total = _randn((n, h), 1, branch).requires_grad_(), _randn((n, h), 6, stream)
        y, total = add_layer_norm(x, res, w, b, EPS, p, seed, call)
        # (dropout's own kernel, which its tests compare with the draws' definition, says
        # what is kept; here the ends of it are looked at)
        keep = dropout(torch.ones((n, h), device="cuda"), p, seed, call) != 0
        m = min(n * h, 4099)
        for first in (0, n * h - m):
            assert torch.equal(keep.view(-1)[first:first + m].cpu(),
                               residual_util.kept((m,), p, seed, call, first))
        scale = keep / (1.0 - p)
        part = x.detach().double() * scale
        want = res.detach().double() + part
        _within(total.detach(), want, 4 * E * part.abs() + E * want.abs() + UNIT[stream] * want.abs()
                + TINY[stream], "total")
        del part, want
        ref = Exact(total, w, b, branch, d_y, d_total)
        d_x, d_res, d_w, d_b = torch.autograd.grad((y, total), (x, res, w, b), (d_y, d_total))
        want = ref.d_s * scale
        _within(d_x, want, ref.tol_s * scale + (4 * E + UNIT[branch]) * want.abs() + TINY[branch],
                "d_x")
    assert y.dtype == branch
    _within(y.detach(), ref.y, ref.tol_y, "y")
    _within(d_res, ref.d_s, ref.tol_s + UNIT[stream] * ref.d_s.abs() + TINY[stream], "d_residual")
    _within(d_w, ref.d_w, ref.tol_w + E * ref.d_w.abs(), "d_weight")
    _within(d_b, ref.d_b, ref.tol_b + E * ref.d_b.abs(), "d_bias")


@pytest.mark.parametrize("stream,branch,h", _widths())
def test_teams(stream, branch, h):
    """Several rows for each team of the largest launch (1,024 threads a CU of 256)."""
    n = max(2600, 256 * 1024 * 5 // 2 // max(8, h // 8) + 3)
    _check(n, h, stream, branch, 0.0, alone=True)
    for p in (0.0, 0.25):
        _check(n, h, stream, branch, p)


@pytest.mark.parametrize("n,h,stream,branch", [(16400, 4096, BF16, BF16), (9001, 4096, F32, BF16),
                                               (9001, 4096, F32, F16), (9001, 4096, F32, F32),
                                               (140001, 520, F16, F16), (50001, 768, F32, BF16),
                                               (7001, 12288, BF16, BF16)])
@pytest.mark.parametrize("how", ["alone", 0.0, 0.1])
def test_past_the_cache(n, h, stream, branch, how):
    """More than 256 MiB of operands each way, rows of whole runs in teams of 64 lanes and
    more: they go past the cache."""
    if how == "alone":
        n = max(n, (260 << 20) // (h * (stream.itemsize + branch.itemsize)))
    operands = n * h * (stream.itemsize + branch.itemsize) * (1 if how == "alone" else 2)
    assert operands > 257 << 20
    _check(n, h, stream, branch, 0.0 if how == "alone" else how, alone=how == "alone")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("wide", [False, True])
def test_dropout_past_the_caches(dtype, wide):
    """More than 32 MiB, alone and onto a residual, of odd length: past the cache."""
    n = 9000011
    stream = F32 if wide else dtype
    x, res = _randn((n,), 1, dtype).requires_grad_(), _randn((n,), 2, stream).requires_grad_()
    g = _randn((n,), 3, stream)
    keep, want, tol = _drop64(x.detach(), res.detach(), 0.3, 17, 3, stream)
    assert n * (dtype.itemsize + stream.itemsize) > 33 << 20
    y = dropout(x, 0.3, 17, 3, residual=res)
    _within(y.detach(), want, tol, "y")
    d_x, = torch.autograd.grad(y, x, g)
    part = torch.where(keep, g.double() / 0.7, 0.0)
    _within(d_x, part, 5 * E * part.abs() + UNIT[dtype] * part.abs() + TINY[dtype], "d_x")
    y = dropout(x, 0.3, 17, 3)
    part = torch.where(keep, x.detach().double() / 0.7, 0.0)
    _within(y.detach(), part, 5 * E * part.abs() + UNIT[dtype] * part.abs() + TINY[dtype], "alone")


@pytest.mark.parametrize("stream,branch", KINDS)
@pytest.mark.parametrize("n,h", [(300, 17000), (300, 17003), (150, 70001)])
def test_rows_that_no_team_holds(n, h, stream, branch):
    """More rows than the parameters' gradients are shared out over."""
    _check(n, h, stream, branch, 0.0, alone=True)
    for p in (0.0, 0.25):
        _check(n, h, stream, branch, p)
