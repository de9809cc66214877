"""The clipped policy loss of sampled tokens, with a KL term.

``policy_loss(logp, old_logp, advantage)`` is what a model that is tuned on its
own answers is trained with: the tokens' log-probabilities are
``-linear_cross_entropy(hidden, weight, target, reduction="none")``, the loss
takes one launch or two for them and its gradient one
(luma_policy_forward / luma_policy_backward in include/luma.h)::

    logp = -luma_amd.linear_cross_entropy(hidden, head.weight, answer, reduction="none")
    loss = luma_amd.policy_loss(logp, old_logp, advantage, mask, ref_logp, kl_weight=0.04)
    loss.backward()

Both directions are ``torch.library`` custom ops, as the other operators' are.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _lib as L
from .loss import _CODES, _REDUCTIONS, _plain
from .residual import _as_rows, _check_device, _check_dtype, _dense, _ld, _ptr, _run

_POLICY_REDUCTIONS = dict(_REDUCTIONS, sequence=L.POLICY_SEQUENCE)

__all__ = ["policy_loss"]


# (by the public function and by the operators, which a recorded graph calls with
# operands that the function has not seen)
def _check_args(logp, old_logp, advantage, mask, ref_logp) -> None:
    _check_dtype("policy_loss", "logp", logp.dtype)
    if logp.dim() < 1:
        raise ValueError("policy_loss: logp has no dimension of tokens")
    for name, t in (("old_logp", old_logp), ("ref_logp", ref_logp)):
        if t is not None and t.dtype != logp.dtype:
            raise ValueError(f"policy_loss: logp is {logp.dtype}, {name} {t.dtype}")
    for name, t in (("old_logp", old_logp), ("ref_logp", ref_logp), ("mask", mask)):
        if t is not None and t.shape != logp.shape:
            raise ValueError(f"policy_loss: {name} {tuple(t.shape)} and logp {tuple(logp.shape)} do "
                             "not match")
    if mask is not None and mask.dtype != torch.bool:
        raise ValueError(f"policy_loss: mask must be bool (got {mask.dtype})")
    if advantage.dtype != torch.float32:
        raise ValueError(f"policy_loss: advantage must be float32 (got {advantage.dtype})")
    if advantage.shape not in (logp.shape, logp.shape[:-1]):
        raise ValueError(f"policy_loss: advantage {tuple(advantage.shape)} is neither one for each "
                         f"token nor one for each sequence of logp {tuple(logp.shape)}")


def _args(logp, old_logp, advantage, mask, ref_logp, share, clip_low, clip_high, kl_weight,
          reduction):
    """(the library's arguments, what has to live until they are used)."""
    each = advantage.dim() == logp.dim()
    lp, old = _as_rows(logp), _as_rows(old_logp)
    ref = None if ref_logp is None else _as_rows(ref_logp)
    m = None if mask is None else _as_rows(mask)
    a = _as_rows(advantage) if each else _dense(advantage)
    return L.PolicyArgs(
        logp=lp.data_ptr(), old_logp=old.data_ptr(), ref_logp=_ptr(ref), advantage=a.data_ptr(),
        mask=_ptr(m), rows=lp.shape[0], length=lp.shape[1], ld_logp=_ld(lp), ld_old=_ld(old),
        ld_ref=0 if ref is None else _ld(ref), ld_advantage=_ld(a) if each else 1,
        ld_mask=0 if m is None else _ld(m), advantage_each=int(each), dtype=_CODES[logp.dtype],
        reduction=reduction, clip_low=clip_low, clip_high=clip_high, kl_weight=kl_weight,
        share=share.data_ptr()), (lp, old, ref, m, a)


@torch.library.custom_op("luma_amd::policy_loss", mutates_args=(), device_types="cuda")
def _forward_op(logp: torch.Tensor, old_logp: torch.Tensor, advantage: torch.Tensor,
                mask: Optional[torch.Tensor], ref_logp: Optional[torch.Tensor], clip_low: float,
                clip_high: float, kl_weight: float, reduction: int,
                figures: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(the loss, its figures or nothing, the rows' shares of a mean)."""
    _check_device("policy_loss", logp=logp, old_logp=old_logp, advantage=advantage, mask=mask,
                  ref_logp=ref_logp)
    _check_args(logp, old_logp, advantage, mask, ref_logp)
    device = logp.device
    rows = 1
    for d in logp.shape[:-1]:
        rows *= d
    none = reduction == L.XENT_NONE

    def new(shape):
        return torch.empty(shape, dtype=torch.float32, device=device)

    loss, share = new(logp.shape if none else ()), new(rows + 1)
    stats = new(L.POLICY_STATS if figures else 0)
    if logp.numel() == 0:
        # (a mean of nothing, as linear_cross_entropy's)
        loss.fill_(0.0 if reduction in (L.XENT_NONE, L.XENT_SUM) else float("nan"))
        stats.fill_(float("nan"))
        stats[3:] = 0.0
        return loss, stats, share.zero_()
    args, live = _args(logp, old_logp, advantage, mask, ref_logp, share, clip_low, clip_high,
                       kl_weight, reduction)
    args.loss, args.stats = loss.data_ptr(), stats.data_ptr() if figures else None
    size = L.load().luma_policy_workspace_bytes(ctypes.byref(args))
    if size < 0:
        L.check(-1, "luma_policy_forward")
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = workspace.data_ptr(), size
    _run("luma_policy_forward", args, device)
    del live
    return loss, stats, share


@_forward_op.register_fake
def _(logp, old_logp, advantage, mask, ref_logp, clip_low, clip_high, kl_weight, reduction, figures):
    rows = 1
    for d in logp.shape[:-1]:
        rows = rows * d

    def new(shape):
        return logp.new_empty(shape, dtype=torch.float32)

    return (new(logp.shape if reduction == L.XENT_NONE else ()),
            new((L.POLICY_STATS if figures else 0,)), new((rows + 1,)))


@torch.library.custom_op("luma_amd::policy_loss_backward", mutates_args=(), device_types="cuda")
def _backward_op(grad: torch.Tensor, logp: torch.Tensor, old_logp: torch.Tensor,
                 advantage: torch.Tensor, mask: Optional[torch.Tensor],
                 ref_logp: Optional[torch.Tensor], share: torch.Tensor, clip_low: float,
                 clip_high: float, kl_weight: float, reduction: int) -> torch.Tensor:
    _check_device("policy_loss", logp=logp, old_logp=old_logp, advantage=advantage, mask=mask,
                  ref_logp=ref_logp, grad=grad, share=share)
    _check_args(logp, old_logp, advantage, mask, ref_logp)
    rows = 1
    for d in logp.shape[:-1]:
        rows *= d
    if grad.shape != (logp.shape if reduction == L.XENT_NONE else ()):
        raise ValueError(f"policy_loss: the gradient {tuple(grad.shape)} is not that of a loss of "
                         f"{tuple(logp.shape)}")
    if share.dtype != torch.float32 or share.shape != (rows + 1,) or not share.is_contiguous():
        raise ValueError(f"policy_loss: share {tuple(share.shape)} is not that of {rows} rows")
    d_logp = torch.empty(logp.shape, dtype=logp.dtype, device=logp.device)
    if logp.numel() == 0:
        return d_logp
    grad = _dense(grad.to(torch.float32))
    args, live = _args(logp, old_logp, advantage, mask, ref_logp, share, clip_low, clip_high,
                       kl_weight, reduction)
    args.grad_loss, args.d_logp = grad.data_ptr(), d_logp.data_ptr()
    _run("luma_policy_backward", args, logp.device)
    del live
    return d_logp


@_backward_op.register_fake
def _(grad, logp, old_logp, advantage, mask, ref_logp, share, clip_low, clip_high, kl_weight,
      reduction):
    return logp.new_empty(logp.shape)


def _setup(ctx, inputs, output):
    (logp, old_logp, advantage, mask, ref_logp, ctx.clip_low, ctx.clip_high, ctx.kl_weight,
     ctx.reduction, _) = inputs
    ctx.save_for_backward(logp, old_logp, advantage, mask, ref_logp, output[2])
    ctx.set_materialize_grads(False)


def _backward(ctx, grad, *_):
    d_logp = None
    if grad is not None and ctx.needs_input_grad[0]:
        logp, old_logp, advantage, mask, ref_logp, share = ctx.saved_tensors
        d_logp = torch.ops.luma_amd.policy_loss_backward(
            grad, logp, old_logp, advantage, mask, ref_logp, share, ctx.clip_low, ctx.clip_high,
            ctx.kl_weight, ctx.reduction)
    return (d_logp,) + (None,) * 9


_forward_op.register_autograd(_backward, setup_context=_setup)


def policy_loss(logp: torch.Tensor, old_logp: torch.Tensor, advantage: torch.Tensor,
                mask: Optional[torch.Tensor] = None, ref_logp: Optional[torch.Tensor] = None, *,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_weight: float = 0.0,
                reduction: str = "mean", return_stats: bool = False
                ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The clipped policy loss of tokens [..., t], float32.

    With r = exp(logp - old_logp) a token's loss is -min(r A, clip(r, 1 -
    clip_low, 1 + clip_high) A), plus, where ``ref_logp`` is given, kl_weight
    (exp(q) - 1 - q) with q = ref_logp - logp (an estimate of the divergence
    from the reference that is never negative; a ``kl_weight`` of 0 leaves it to
    the figures alone, whatever it is).  ``advantage`` A is float32, one
    for each token or one for each sequence (logp's shape without its last
    dimension); the log-probabilities are float32, bfloat16 or float16, all of
    one type.  The gradient is logp's alone: the others are constants, whatever
    they require.  Where both products are the same the gradient is the
    unclipped one's.

    ``mask`` (bool): the tokens that count.  What stands in the others' places,
    infinities and NaN among it, reaches neither the loss nor the gradient,
    which is 0 there.  ``reduction``: "mean" over the tokens, "sequence" (the
    mean over the sequences that have tokens of each one's mean), "sum" or
    "none"; a mean over nothing is NaN.

    ``return_stats``: also four float32 numbers for a log, over the tokens that
    count: the share whose ratio was clipped, the mean of the KL term (without
    its weight; 0 without ``ref_logp``), that of r - 1 - log r (how far the
    policy has moved), and how many tokens there are.  Rows of more than 1,024
    tokens: 2^22 at most.  The gradient cannot be differentiated again (that
    raises).
    """
    code = _POLICY_REDUCTIONS.get(reduction)
    if code is None:
        raise ValueError(f"Invalid reduction: {reduction!r}. Expected 'none', 'sum', 'mean' or "
                         "'sequence'")
    clip_low, clip_high, kl_weight = float(clip_low), float(clip_high), float(kl_weight)
    if not 0.0 <= clip_low <= 1.0 or not clip_high >= 0.0 or kl_weight != kl_weight:
        raise ValueError(f"policy_loss: clip_low must be in [0, 1], clip_high not negative and "
                         f"kl_weight a number (got {clip_low}, {clip_high}, {kl_weight})")
    compiling = torch.compiler.is_compiling()
    if not compiling and _plain(*(t for t in (logp, old_logp, advantage, mask, ref_logp)
                                  if t is not None)):
        host = L.host_calls()
        out = None if host is None else host.policy_loss(logp, old_logp, advantage, mask, ref_logp,
                                                         clip_low, clip_high, kl_weight, code,
                                                         return_stats)
        if out is not None:
            return out
    _check_args(logp, old_logp, advantage, mask, ref_logp)
    if not compiling:
        _check_device("policy_loss", logp=logp, old_logp=old_logp, advantage=advantage, mask=mask,
                      ref_logp=ref_logp)
    old_logp, advantage = old_logp.detach(), advantage.detach()
    ref_logp = None if ref_logp is None else ref_logp.detach()
    loss, stats, _ = torch.ops.luma_amd.policy_loss(logp, old_logp, advantage, mask, ref_logp,
                                                    clip_low, clip_high, kl_weight, code,
                                                    return_stats)
    return (loss, stats.detach()) if return_stats else loss
