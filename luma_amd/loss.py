"""Cross entropy of a vocabulary head's logits, without the logits.

``linear_cross_entropy(hidden, weight, target)`` is
``F.cross_entropy(F.linear(hidden, weight), target)``, the loss that the
reference's benchmark trains on (benchmarks/bench_nanogpt.py), for a head of
any size: the logits are formed tile by tile on the matrix cores and consumed
there, and the backward forms them again, a piece of the vocabulary at a time
(luma_xent_forward / luma_xent_backward in include/luma.h).  Both directions
are ``torch.library`` custom ops, so ``torch.compile(fullgraph=True)``, ``make_fx``
and ``torch.jit.trace`` record them, and they do no host synchronisation (an
eager call that nothing records goes through the host module, to the same
kernels)::

    loss = luma_amd.linear_cross_entropy(hidden, head.weight, target)
    loss.backward()
"""

from __future__ import annotations

import ctypes
from typing import Tuple

import torch

from . import _lib as L

_CODES = {torch.float32: L.GRAD_F32, torch.bfloat16: L.GRAD_BF16, torch.float16: L.GRAD_F16}
_REDUCTIONS = {"none": L.XENT_NONE, "sum": L.XENT_SUM, "mean": L.XENT_MEAN}

__all__ = ["linear_cross_entropy"]


def _check(hidden, weight, target) -> None:
    for name, t in (("hidden", hidden), ("weight", weight), ("target", target)):
        if not t.is_cuda:
            raise RuntimeError(f"linear_cross_entropy: {name} must be on a ROCm GPU; got "
                               f"{t.device}")
        if t.device != hidden.device:
            raise ValueError(f"linear_cross_entropy: {name} is on {t.device}, hidden on "
                             f"{hidden.device}")


def _check_types(hidden, weight, target) -> None:
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_cross_entropy: hidden {tuple(hidden.shape)} and weight "
                         f"{tuple(weight.shape)} do not match")
    if hidden.dtype not in _CODES:
        raise ValueError(f"linear_cross_entropy: dtype {hidden.dtype} is not "
                         "float32/bfloat16/float16")
    if weight.dtype != hidden.dtype:
        raise ValueError(f"linear_cross_entropy: hidden is {hidden.dtype}, weight {weight.dtype} "
                         "(torch.autocast casts both)")
    if target.dtype != torch.int64:
        raise ValueError(f"linear_cross_entropy: target must be int64 (got {target.dtype})")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: target {tuple(target.shape)} does not match "
                         f"hidden {tuple(hidden.shape)}")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError("linear_cross_entropy: the vocabulary and the hidden states must not be "
                         "empty")


def _check_operands(hidden, weight, target, **more) -> None:
    """What an operator is called with (by a recorded graph, with operands that the
    public function has not seen)."""
    _check(hidden, weight, target)
    for name, t in more.items():
        if t.device != hidden.device:
            raise ValueError(f"linear_cross_entropy: {name} is on {t.device}, hidden on "
                             f"{hidden.device}")
    if hidden.dim() != 2:
        raise ValueError(f"linear_cross_entropy: hidden {tuple(hidden.shape)} are not rows")
    _check_types(hidden, weight, target)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy, with elements of a row next to each other and rows apart."""
    if t.is_neg() or t._is_zerotensor() or (t.shape[1] > 1 and t.stride(1) != 1) or (
            t.shape[0] > 1 and not t.shape[1] <= t.stride(0) <= 1 << 21):
        return t.contiguous()
    return t


def _args(hidden, weight, target, stats, ignore_index, reduction) -> L.XentArgs:
    n, h = hidden.shape
    return L.XentArgs(
        hidden=hidden.data_ptr(), weight=weight.data_ptr(), target=target.data_ptr(), n=n, h=h,
        v=weight.shape[0], ld_hidden=hidden.stride(0) if n > 1 else h,
        ld_weight=weight.stride(0) if weight.shape[0] > 1 else h, ignore_index=ignore_index,
        dtype=_CODES[hidden.dtype], reduction=reduction, stats=stats.data_ptr())


def _call(name: str, args: L.XentArgs, device) -> None:
    lib = L.load()
    backward = name == "luma_xent_backward"
    size = lib.luma_xent_workspace_bytes(ctypes.byref(args), backward)
    if size < 0:
        L.check(-1, name)
    workspace = torch.empty(max(size, 1), dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = workspace.data_ptr(), size
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        L.check(getattr(lib, name)(ctypes.byref(args), stream), name)


@torch.library.custom_op("luma_amd::linear_cross_entropy", mutates_args=(), device_types="cuda")
def _forward_op(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                ignore_index: int, reduction: int) -> Tuple[torch.Tensor, torch.Tensor]:
    _check_operands(hidden, weight, target)
    n, device = hidden.shape[0], hidden.device
    loss = torch.empty((n,) if reduction == L.XENT_NONE else (), dtype=torch.float32,
                       device=device)
    if n == 0:
        loss.fill_(float("nan") if reduction == L.XENT_MEAN else 0.0)
        return loss, torch.zeros(1, dtype=torch.float32, device=device)
    stats = torch.empty(2 * n + 1, dtype=torch.float32, device=device)
    hidden, weight, target = _rows(hidden), _rows(weight), target.contiguous()
    args = _args(hidden, weight, target, stats, ignore_index, reduction)
    args.loss = loss.data_ptr()
    _call("luma_xent_forward", args, device)
    return loss, stats


@_forward_op.register_fake
def _(hidden, weight, target, ignore_index, reduction):
    n = hidden.shape[0]
    loss = hidden.new_empty((n,) if reduction == L.XENT_NONE else (), dtype=torch.float32)
    return loss, hidden.new_empty((2 * n + 1,), dtype=torch.float32)


@torch.library.custom_op("luma_amd::linear_cross_entropy_backward", mutates_args=(),
                         device_types="cuda")
def _backward_op(grad: torch.Tensor, hidden: torch.Tensor, weight: torch.Tensor,
                 target: torch.Tensor, stats: torch.Tensor, ignore_index: int, reduction: int,
                 want_hidden: bool, want_weight: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    _check_operands(hidden, weight, target, grad=grad, stats=stats)
    n, device = hidden.shape[0], hidden.device
    if grad.shape != ((n,) if reduction == L.XENT_NONE else ()):
        raise ValueError(f"linear_cross_entropy: the gradient {tuple(grad.shape)} is not that of a "
                         f"loss of {n} tokens")
    if stats.dtype != torch.float32 or stats.shape != (2 * n + 1,) or not stats.is_contiguous():
        raise ValueError(f"linear_cross_entropy: stats {tuple(stats.shape)} are not those of {n} "
                         "tokens")
    d_hidden = torch.empty(hidden.shape if want_hidden else (0,), dtype=hidden.dtype,
                           device=device)
    d_weight = torch.empty(weight.shape if want_weight else (0,), dtype=weight.dtype,
                           device=device)
    if n == 0:
        return d_hidden, d_weight.zero_()
    hidden, weight, target = _rows(hidden), _rows(weight), target.contiguous()
    grad = grad.to(torch.float32).contiguous()
    args = _args(hidden, weight, target, stats, ignore_index, reduction)
    args.grad_loss = grad.data_ptr()
    args.d_hidden = d_hidden.data_ptr() if want_hidden else None
    args.d_weight = d_weight.data_ptr() if want_weight else None
    _call("luma_xent_backward", args, device)
    return d_hidden, d_weight


@_backward_op.register_fake
def _(grad, hidden, weight, target, stats, ignore_index, reduction, want_hidden, want_weight):
    return (hidden.new_empty(hidden.shape if want_hidden else (0,)),
            weight.new_empty(weight.shape if want_weight else (0,)))


def _setup(ctx, inputs, output):
    hidden, weight, target, ctx.ignore_index, ctx.reduction = inputs
    ctx.save_for_backward(hidden, weight, target, output[1])
    ctx.set_materialize_grads(False)


def _backward(ctx, grad, _):
    hidden, weight, target, stats = ctx.saved_tensors
    want_hidden, want_weight = ctx.needs_input_grad[:2]
    if grad is None or not (want_hidden or want_weight):
        return None, None, None, None, None
    d_hidden, d_weight = torch.ops.luma_amd.linear_cross_entropy_backward(
        grad, hidden, weight, target, stats, ctx.ignore_index, ctx.reduction, want_hidden,
        want_weight)
    return (d_hidden if want_hidden else None, d_weight if want_weight else None, None, None,
            None)


_forward_op.register_autograd(_backward, setup_context=_setup)


def _plain(*tensors) -> bool:
    """Whether the host module may take the call: nothing records or watches the
    operators called (a tracer or a dispatch mode would see the allocation of
    the module's outputs, and not the kernels that fill them), and no tensor is
    of a subclass with a dispatch of its own, or one of torch.func's."""
    return (torch._C._len_torch_dispatch_stack() == 0
            and torch._ops._len_torch_dispatch_stack_pre_dispatch() == 0
            and torch._C._get_tracing_state() is None
            and not torch._C._are_functorch_transforms_active()
            and all(type(t) is torch.Tensor or type(t) is torch.nn.Parameter for t in tensors))


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """``F.cross_entropy`` of ``hidden @ weight.T`` against ``target``, float32.

    ``hidden`` [..., h] and ``weight`` [v, h] are float32, bfloat16 or float16
    on one GPU, of one type (under ``torch.autocast`` both are cast to its
    type, as a linear layer's operands are); ``target`` [...] is int64.  The
    products are summed in float32, the softmax is float32; the gradients have
    the operands' type, and the logits' gradient is rounded to it between its
    two products.  ``reduction``: "mean" (over the targets that are not
    ``ignore_index``; NaN if there are none), "sum" or "none" (a loss per
    token, the target's shape).  A target that is neither a word nor
    ``ignore_index`` makes its loss NaN (nothing is read for it); torch stops
    the program there.  The gradients cannot be differentiated again (that raises).
    """
    code = _REDUCTIONS.get(reduction)
    if code is None:
        raise ValueError(f"Invalid reduction: {reduction!r}. Expected 'none', 'sum' or 'mean'")
    if hidden.is_cuda and torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        hidden, weight = hidden.to(dtype), weight.to(dtype)
    compiling = torch.compiler.is_compiling()
    if not compiling and _plain(hidden, weight, target):
        host = L.host_calls()
        loss = None if host is None else host.xent(hidden, weight, target, ignore_index, code)
        if loss is not None:
            return loss
    _check_types(hidden, weight, target)
    if not compiling:
        _check(hidden, weight, target)
    shape = target.shape
    if len(shape) != 1:
        hidden, target = hidden.reshape(-1, hidden.shape[-1]), target.reshape(-1)
    loss, _ = torch.ops.luma_amd.linear_cross_entropy(hidden, weight, target, ignore_index, code)
    return loss.view(shape) if code == L.XENT_NONE and len(shape) != 1 else loss
