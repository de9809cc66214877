"""The residual stream of a model's blocks: layer normalisation, dropout, and
both at a block's border, forward and backward, in one kernel each way.

The reference's benchmark runs torch's layers there
(benchmarks/bench_nanogpt.py).  ``layer_norm`` is ``F.layer_norm`` over the last
dimension, ``dropout`` draws its mask from a counter-based generator and never
stores it, and ``add_layer_norm`` adds a branch's output (dropped out) to the
stream and normalises the sum for the next branch (luma_layer_norm_forward /
_backward, luma_dropout in include/luma.h)::

    y = luma_amd.layer_norm(x, norm.weight, norm.bias, norm.eps)
    y, x = luma_amd.add_layer_norm(branch(y), x, norm.weight, norm.bias, norm.eps,
                                   p=0.1, seed=step, call=layer)

Both directions are ``torch.library`` custom ops, so
``torch.compile(fullgraph=True)``, ``make_fx`` and ``torch.jit.trace`` record
them, and they do no host synchronisation (an eager call that nothing records
goes through the host module, to the same kernels).
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _lib as L
from .loss import _CODES, _plain

_TYPES = {code: dtype for dtype, code in _CODES.items()}

__all__ = ["add_layer_norm", "dropout", "layer_norm"]


# -- what is passed to the library ----------------------------------------------


def _resolved(t: torch.Tensor) -> torch.Tensor:
    """t with memory that holds its values."""
    if t._is_zerotensor():
        return torch.zeros(t.shape, dtype=t.dtype, device=t.device)
    return t.resolve_neg()


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else _resolved(t).contiguous()


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy, as rows of its last dimension, elements of a row next to
    each other."""
    t = _resolved(t)
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t.contiguous() if t.shape[1] > 1 and t.stride(1) != 1 else t


def _ld(rows: torch.Tensor) -> int:
    return rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _drop(seed_at, p, seed, call) -> L.Dropout:
    return L.Dropout(seed_at=_ptr(seed_at), seed=seed & (1 << 64) - 1, p=p, call=call)


def _run(name: str, args, device) -> None:
    lib = L.load()
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        L.check(getattr(lib, name)(ctypes.byref(args), stream), name)


# -- checks -----------------------------------------------------------------------
# (by the public functions, and by the operators: a recorded graph calls those with
# operands that the functions have not seen)


def _check_device(what: str, **tensors) -> None:
    first = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{what}: {name} must be on a ROCm GPU; got {t.device}")
        if first is not None and t.device != first[1].device:
            raise ValueError(f"{what}: {name} is on {t.device}, {first[0]} on {first[1].device}")
        first = first or (name, t)


def _check_dtype(what: str, name: str, dtype) -> None:
    if dtype not in _CODES:
        raise ValueError(f"{what}: {name} {dtype} is not float32/bfloat16/float16")


def _check_stream(what: str, residual, x) -> None:
    _check_dtype(what, "residual", residual.dtype)
    if residual.shape != x.shape:
        raise ValueError(f"{what}: residual {tuple(residual.shape)} and x {tuple(x.shape)} do not "
                         "match")
    if residual.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"{what}: residual is {residual.dtype}, x {x.dtype} (the residual has "
                         "x's type or float32)")


def _check_seed(what: str, seed) -> None:
    if seed is not None and (seed.dtype != torch.int64 or seed.numel() != 1):
        raise ValueError(f"{what}: a seed on the device is one int64 number (got "
                         f"{tuple(seed.shape)} {seed.dtype})")


def _draws(what: str, p, seed, call) -> Tuple[float, Optional[torch.Tensor], int, int]:
    """(p, the seed's tensor or None, the seed as a signed 64-bit number, call)."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: p must be in [0, 1] (got {p})")
    call = int(call)
    if not 0 <= call < 1 << 32:
        raise ValueError(f"{what}: call must be in [0, 2^32) (got {call})")
    if isinstance(seed, torch.Tensor):
        _check_seed(what, seed)
        return p, seed, 0, call
    seed = int(seed)
    if not -1 << 63 <= seed < 1 << 64:
        raise ValueError(f"{what}: seed must fit 64 bits (got {seed})")
    return p, None, seed - (1 << 64) if seed >= 1 << 63 else seed, call


def _check_norm(what: str, x, residual, weight, bias, eps, branch) -> None:
    _check_dtype(what, "x", x.dtype)
    _check_dtype(what, "dtype", branch)
    if residual is not None:
        _check_stream(what, residual, x)
    if branch != x.dtype and (residual is not None or x.dtype != torch.float32):
        raise ValueError(f"{what}: dtype {branch} of a result from {x.dtype} (it is x's, or a "
                         "16-bit one for a float32 x)")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{what}: x {tuple(x.shape)} has no rows of elements")
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must not be negative (got {eps})")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != x.shape[-1:]:
            raise ValueError(f"{what}: {name} {tuple(t.shape)} and x {tuple(x.shape)} do not match")
        if t.dtype not in (torch.float32, branch):
            raise ValueError(f"{what}: {name} is {t.dtype}, the result {branch} (weight and bias "
                             "have its type or float32)")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"{what}: weight is {weight.dtype}, bias {bias.dtype}")


# -- dropout ----------------------------------------------------------------------


def _check_dropout(x, residual) -> None:
    _check_dtype("dropout", "x", x.dtype)
    if residual is not None:
        _check_stream("dropout", residual, x)


def _dropout_call(x, residual, y, seed_at, p, seed, call) -> None:
    if x.numel() == 0:
        return
    x, residual = _dense(x), _dense(residual)
    _run("luma_dropout", L.DropoutArgs(
        x=x.data_ptr(), residual=_ptr(residual), y=y.data_ptr(), numel=x.numel(),
        in_type=_CODES[x.dtype], out_type=_CODES[y.dtype], drop=_drop(seed_at, p, seed, call)),
        x.device)


@torch.library.custom_op("luma_amd::dropout", mutates_args=(), device_types="cuda")
def _dropout_op(x: torch.Tensor, residual: Optional[torch.Tensor],
                seed_at: Optional[torch.Tensor], p: float, seed: int, call: int) -> torch.Tensor:
    _check_device("dropout", x=x, residual=residual, seed=seed_at)
    _check_seed("dropout", seed_at)
    _check_dropout(x, residual)
    y = torch.empty(x.shape, dtype=(x if residual is None else residual).dtype, device=x.device)
    _dropout_call(x, residual, y, seed_at, p, seed, call)
    return y


@_dropout_op.register_fake
def _(x, residual, seed_at, p, seed, call):
    return x.new_empty(x.shape, dtype=(x if residual is None else residual).dtype)


@torch.library.custom_op("luma_amd::dropout_backward", mutates_args=(), device_types="cuda")
def _dropout_backward_op(grad: torch.Tensor, seed_at: Optional[torch.Tensor], p: float, seed: int,
                         call: int, code: int) -> torch.Tensor:
    _check_device("dropout", grad=grad, seed=seed_at)
    _check_dtype("dropout", "the gradient", grad.dtype)
    _check_seed("dropout", seed_at)
    d_x = torch.empty(grad.shape, dtype=_TYPES[code], device=grad.device)
    _dropout_call(grad, None, d_x, seed_at, p, seed, call)
    return d_x


@_dropout_backward_op.register_fake
def _(grad, seed_at, p, seed, call, code):
    return grad.new_empty(grad.shape, dtype=_TYPES[code])


def _dropout_setup(ctx, inputs, output):
    x, _, seed_at, ctx.p, ctx.seed, ctx.call = inputs
    ctx.code = _CODES[x.dtype]
    ctx.save_for_backward(seed_at)
    ctx.set_materialize_grads(False)


def _dropout_grad(ctx, grad):
    d_x = None
    if grad is not None and ctx.needs_input_grad[0]:
        d_x = torch.ops.luma_amd.dropout_backward(grad, ctx.saved_tensors[0], ctx.p, ctx.seed,
                                                  ctx.call, ctx.code)
    return d_x, grad if ctx.needs_input_grad[1] else None, None, None, None, None


_dropout_op.register_autograd(_dropout_grad, setup_context=_dropout_setup)


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], call: int = 0,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` with each element dropped with probability ``p`` and the others
    scaled by 1 / (1 - p); with ``residual``, that added to it.

    The mask follows from ``seed``, ``call`` and the element's index alone, and
    the backward draws it again: nothing is stored.  ``seed`` is a number of 64
    bits or a one-element int64 tensor on x's device, which the kernels read
    (under a captured graph a program advances it between the replays; it must
    not be written between a forward and its backward); ``call`` (32 bits) tells
    the places of a model that share a seed from each other.  Draws are those
    of Philox4x32-10, 32 bits an element (LumaDropout in include/luma.h says
    which): the same on every GPU, in every type, and for every way of calling.
    A dropped element is 0 whatever it held.  ``p`` = 0 (evaluation) draws
    nothing.

    ``x`` is float32, bfloat16 or float16; ``residual`` has its shape and its
    type or float32, and the result the residual's type (x's without one); the
    sum is formed in float32; at most 2^34 elements.  The gradients cannot be
    differentiated again (that raises).
    """
    p, seed_at, seed, call = _draws("dropout", p, seed, call)
    compiling = torch.compiler.is_compiling()
    if not compiling and _plain(*(t for t in (x, residual, seed_at) if t is not None)):
        host = L.host_calls()
        y = None if host is None else host.dropout(x, residual, seed_at, p, seed, call)
        if y is not None:
            return y
    _check_dropout(x, residual)
    if not compiling:
        _check_device("dropout", x=x, residual=residual, seed=seed_at)
    return torch.ops.luma_amd.dropout(x, residual, seed_at, p, seed, call)


# -- layer normalisation ------------------------------------------------------------


def _norm_args(x, weight, bias, stream, branch, param, seed_at, p, seed, call) -> L.LayerNormArgs:
    return L.LayerNormArgs(
        weight=_ptr(weight), bias=_ptr(bias), n=x.shape[0], h=x.shape[1],
        stream=stream, branch=branch, param=param, drop=_drop(seed_at, p, seed, call))


def _param_code(weight, bias) -> int:
    for t in (weight, bias):
        if t is not None:
            return _CODES[t.dtype]
    return L.GRAD_F32


@torch.library.custom_op("luma_amd::layer_norm", mutates_args=(), device_types="cuda")
def _norm_op(x: torch.Tensor, residual: Optional[torch.Tensor], weight: Optional[torch.Tensor],
             bias: Optional[torch.Tensor], seed_at: Optional[torch.Tensor], eps: float, p: float,
             seed: int, call: int,
             branch: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, the sum or nothing, each row's mean and 1 / deviation)."""
    what = "layer_norm" if residual is None else "add_layer_norm"
    _check_device(what, x=x, residual=residual, weight=weight, bias=bias, seed=seed_at)
    _check_seed(what, seed_at)
    _check_norm(what, x, residual, weight, bias, eps, _TYPES.get(branch))
    like, device = x if residual is None else residual, x.device
    rows = x.numel() // x.shape[-1]
    y = torch.empty(x.shape, dtype=_TYPES[branch], device=device)
    total = torch.empty((0,) if residual is None else x.shape, dtype=like.dtype, device=device)
    stats = torch.empty(2 * rows, dtype=torch.float32, device=device)
    if rows == 0:
        return y, total, stats
    xs, rs = _as_rows(x), None if residual is None else _as_rows(residual)
    w, b = _dense(weight), _dense(bias)
    args = _norm_args(xs, w, b, _CODES[like.dtype], branch, _param_code(weight, bias), seed_at, p,
                      seed, call)
    args.x, args.ld_x, args.eps = xs.data_ptr(), _ld(xs), eps
    args.y, args.stats = y.data_ptr(), stats.data_ptr()
    if rs is not None:
        args.residual, args.ld_residual, args.total = rs.data_ptr(), _ld(rs), total.data_ptr()
    _run("luma_layer_norm_forward", args, device)
    return y, total, stats


@_norm_op.register_fake
def _(x, residual, weight, bias, seed_at, eps, p, seed, call, branch):
    like = x if residual is None else residual
    rows = 1
    for d in x.shape[:-1]:
        rows = rows * d
    return (x.new_empty(x.shape, dtype=_TYPES[branch]),
            x.new_empty((0,) if residual is None else x.shape, dtype=like.dtype),
            x.new_empty((2 * rows,), dtype=torch.float32))


@torch.library.custom_op("luma_amd::layer_norm_backward", mutates_args=(), device_types="cuda")
def _norm_backward_op(d_y: torch.Tensor, d_total: Optional[torch.Tensor], s: torch.Tensor,
                      weight: Optional[torch.Tensor], stats: torch.Tensor,
                      seed_at: Optional[torch.Tensor], p: float, seed: int, call: int, branch: int,
                      param: int, adds: bool, want_x: bool, want_residual: bool, want_weight: bool,
                      want_bias: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor,
                                                torch.Tensor]:
    """The gradients of x, the residual, weight and bias (empty ones where not
    wanted); s is the sum, or x without a residual."""
    device, h = s.device, s.shape[-1]
    what = "add_layer_norm" if adds else "layer_norm"
    _check_device(what, sum=s, d_y=d_y, d_total=d_total, weight=weight, stats=stats, seed=seed_at)
    _check_seed(what, seed_at)
    _check_dtype(what, "the sum", s.dtype)
    for name, t in (("d_y", d_y), ("d_total", d_total)):
        if t is not None and t.shape != s.shape:
            raise ValueError(f"{what}: {name} {tuple(t.shape)} and the sum {tuple(s.shape)} do not "
                             "match")
    if weight is not None and (weight.shape != s.shape[-1:] or weight.dtype != _TYPES.get(param)):
        raise ValueError(f"{what}: weight {tuple(weight.shape)} {weight.dtype} does not match the sum "
                         f"{tuple(s.shape)}")
    if (stats.dtype != torch.float32 or stats.numel() * h != 2 * s.numel()
            or not stats.is_contiguous()):
        raise ValueError(f"{what}: stats {tuple(stats.shape)} are not those of rows "
                         f"{tuple(s.shape)}")

    def new(wanted, shape, dtype):
        return torch.empty(shape if wanted else (0,), dtype=dtype, device=device)

    d_x = new(want_x, s.shape, _TYPES[branch] if adds else s.dtype)
    d_residual = new(want_residual, s.shape, s.dtype)
    d_weight, d_bias = new(want_weight, (h,), _TYPES[param]), new(want_bias, (h,), _TYPES[param])
    if s.numel() == 0:
        return d_x, d_residual, d_weight.zero_(), d_bias.zero_()
    ss, w = _as_rows(s), _dense(weight)
    dy, dt = _dense(d_y.to(_TYPES[branch])), None if d_total is None else _dense(d_total.to(s.dtype))
    args = _norm_args(ss, w, None, _CODES[s.dtype], branch, param, seed_at, p, seed, call)
    args.x, args.ld_x = ss.data_ptr(), _ld(ss)
    args.total = ss.data_ptr() if adds else None
    args.stats, args.d_y, args.d_total = stats.data_ptr(), dy.data_ptr(), _ptr(dt)
    args.d_x = d_x.data_ptr() if want_x else None
    args.d_residual = d_residual.data_ptr() if want_residual else None
    args.d_weight = d_weight.data_ptr() if want_weight else None
    args.d_bias = d_bias.data_ptr() if want_bias else None
    workspace = None
    if want_weight or want_bias:
        size = L.load().luma_layer_norm_workspace_bytes(ctypes.byref(args))
        if size < 0:
            L.check(-1, "luma_layer_norm_backward")
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), size
    _run("luma_layer_norm_backward", args, device)
    return d_x, d_residual, d_weight, d_bias


@_norm_backward_op.register_fake
def _(d_y, d_total, s, weight, stats, seed_at, p, seed, call, branch, param, adds, want_x,
      want_residual, want_weight, want_bias):
    h = s.shape[-1]

    def new(wanted, shape, dtype):
        return s.new_empty(shape if wanted else (0,), dtype=dtype)

    return (new(want_x, s.shape, _TYPES[branch] if adds else s.dtype),
            new(want_residual, s.shape, s.dtype), new(want_weight, (h,), _TYPES[param]),
            new(want_bias, (h,), _TYPES[param]))


def _norm_setup(ctx, inputs, output):
    x, residual, weight, bias, seed_at, _, ctx.p, ctx.seed, ctx.call, ctx.branch = inputs
    _, total, stats = output
    ctx.adds, ctx.param = residual is not None, _param_code(weight, bias)
    ctx.save_for_backward(total if ctx.adds else x, weight, stats, seed_at)
    ctx.set_materialize_grads(False)


def _norm_grad(ctx, d_y, d_total, _):
    s, weight, stats, seed_at = ctx.saved_tensors
    want = list(ctx.needs_input_grad[:4])
    if not ctx.adds:
        d_total = None
    if (d_y is None and d_total is None) or not any(want):
        return (None,) * 10
    # (without draws the sum's gradient is that of both)
    one = ctx.adds and ctx.p == 0.0 and _CODES[s.dtype] == ctx.branch
    if d_y is None:
        # The sum alone was used: its norm has no part in the gradients, whether those of
        # its rows are numbers or not.
        d_total = d_x = d_total.to(s.dtype)
        if want[0] and not one:
            d_x = torch.ops.luma_amd.dropout_backward(d_total, seed_at, ctx.p, ctx.seed, ctx.call,
                                                      ctx.branch)
        zero = s.new_zeros(s.shape[-1:], dtype=_TYPES[ctx.param])
        got = (d_x, d_total, zero, zero)
        return tuple(g if w else None for g, w in zip(got, want)) + (None,) * 6
    want_x, want_residual = want[0] and not one, want[1] or (one and want[0])
    d_x, d_residual, d_weight, d_bias = torch.ops.luma_amd.layer_norm_backward(
        d_y, d_total, s, weight, stats, seed_at, ctx.p, ctx.seed, ctx.call, ctx.branch, ctx.param,
        ctx.adds, want_x, want_residual, want[2], want[3])
    got = (d_residual if one else d_x, d_residual, d_weight, d_bias)
    return tuple(g if w else None for g, w in zip(got, want)) + (None,) * 6


_norm_op.register_autograd(_norm_grad, setup_context=_norm_setup)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``F.layer_norm(x, x.shape[-1:], weight, bias, eps)`` in one kernel each way.

    ``x`` [..., h] is float32, bfloat16 or float16.  ``dtype`` is the result's
    type: x's (the default), or a 16-bit one for a float32 x, as the layer
    behind it reads under mixed precision; ``torch.autocast`` changes nothing
    here.  ``weight`` and ``bias`` [h] (either may be left out) are float32 or of
    the result's type, both the same.  Mean, deviation and the sums of the
    gradients are float32, the result and each gradient are rounded once, and
    the weight's gradient is the same on every call.  At most 2^31 - 1 rows, of
    2^24 elements.  The gradients cannot be differentiated again (that raises).
    """
    dtype = x.dtype if dtype is None else dtype
    code = _CODES.get(dtype, -1)
    compiling = torch.compiler.is_compiling()
    if not compiling and _plain(*(t for t in (x, weight, bias) if t is not None)):
        host = L.host_calls()
        y = None if host is None else host.layer_norm(x, None, weight, bias, None, eps, 0.0, 0, 0,
                                                      code)
        if y is not None:
            return y
    _check_norm("layer_norm", x, None, weight, bias, eps, dtype)
    if not compiling:
        _check_device("layer_norm", x=x, weight=weight, bias=bias)
    return torch.ops.luma_amd.layer_norm(x, None, weight, bias, None, eps, 0.0, 0, 0, code)[0]


def add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5, p: float = 0.0,
                   seed: Union[int, torch.Tensor] = 0,
                   call: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """A block's border: ``total = residual + dropout(x)`` and ``y =
    layer_norm(total)``; returns ``(y, total)``.

    ``x`` [..., h], a branch's output, is float32, bfloat16 or float16, and so is
    ``y``; ``residual`` and ``total``, the stream, have its type or float32.
    ``p``, ``seed`` and ``call`` are ``dropout``'s (the same mask), weight, bias
    and eps ``layer_norm``'s.  ``total`` is rounded to the stream's type before
    its norm is taken: the results are those of ``dropout(x, p, seed, call,
    residual)`` and of ``layer_norm`` of that, but for float16's double
    roundings.  A ``y`` that goes unused leaves the sum's gradients, and zeros
    for weight and bias.  The gradients cannot be differentiated again (that
    raises).
    """
    p, seed_at, seed, call = _draws("add_layer_norm", p, seed, call)
    code = _CODES.get(x.dtype, -1)
    compiling = torch.compiler.is_compiling()
    if not compiling and _plain(*(t for t in (x, residual, weight, bias, seed_at)
                                  if t is not None)):
        host = L.host_calls()
        out = None if host is None else host.layer_norm(x, residual, weight, bias, seed_at, eps, p,
                                                        seed, call, code)
        if out is not None:
            return out
    _check_norm("add_layer_norm", x, residual, weight, bias, eps, x.dtype)
    if not compiling:
        _check_device("add_layer_norm", x=x, residual=residual, weight=weight, bias=bias,
                      seed=seed_at)
    y, total, _ = torch.ops.luma_amd.layer_norm(x, residual, weight, bias, seed_at, eps, p, seed,
                                                call, code)
    return y, total
