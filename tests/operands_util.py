"""Operands of the operators beside the step, by name and in the operators' order, that
fit each other, and changes of them that do not."""

import torch

DEVICE = "cuda"


def tensor(*shape, dtype=torch.float32):
    return torch.full(shape, 0.5, device=DEVICE).to(dtype)


BF16, F16, F64 = torch.bfloat16, torch.float16, torch.float64


def _width(*s):
    return tensor(s[-1])


def _rows(*s):
    return tensor(s[0])


def _mask(*s):
    return tensor(*s) > 0


def _words(*s):
    return torch.zeros(s[0], dtype=torch.int64, device=DEVICE)


# Operands (by name, in the operators' order) that fit.
CALLS = {
    "dropout": dict(x=tensor, residual=tensor, seed=None, p=0.5, number=1, call=0),
    "dropout_backward": dict(grad=tensor, seed=None, p=0.5, number=1, call=0, code=0),
    "layer_norm": dict(x=tensor, residual=tensor, weight=_width, bias=_width, seed=None, eps=1e-5,
                       p=0.5, number=1, call=0, branch=0),
    "layer_norm_backward": dict(d_y=tensor, d_total=tensor, s=tensor, weight=_width,
                                stats=lambda *s: tensor(2 * s[0]), seed=None, p=0.5, number=1,
                                call=0, branch=0, param=0, adds=True, want_x=True,
                                want_residual=True, want_weight=True, want_bias=True),
    "policy_loss": dict(logp=tensor, old=tensor, advantage=_rows, mask=_mask, ref=tensor, low=0.2,
                        high=0.2, kl=0.1, reduction=2, figures=True),
    "policy_loss_backward": dict(grad=lambda *s: tensor(), logp=tensor, old=tensor, advantage=_rows,
                                 mask=_mask, ref=tensor, share=lambda *s: tensor(s[0] + 1), low=0.2,
                                 high=0.2, kl=0.1, reduction=2),
    "linear_cross_entropy": dict(hidden=tensor, weight=lambda *s: tensor(50, s[1]), target=_words,
                                 ignore=-100, reduction=2),
    "linear_cross_entropy_backward": dict(grad=lambda *s: tensor(), hidden=tensor,
                                          weight=lambda *s: tensor(50, s[1]), target=_words,
                                          stats=lambda *s: tensor(2 * s[0] + 1), ignore=-100,
                                          reduction=2, want_hidden=True, want_weight=True),
}
SEEDS = [dict(seed=torch.zeros(1, dtype=torch.int32)), dict(seed=torch.zeros(2, dtype=torch.int64)),
         dict(seed=torch.zeros(0, dtype=torch.int64))]
BAD = {
    "dropout": [dict(residual=(5, 24)), dict(residual=(6, 23)), dict(residual=BF16), dict(x=F64),
                *SEEDS],
    "dropout_backward": [dict(grad=F64), *SEEDS],
    "layer_norm": [dict(residual=(5, 24)), dict(residual=(6, 20)), dict(residual=BF16), dict(x=BF16),
                   dict(x=F64), dict(weight=(20,)), dict(bias=(20,)), dict(weight=BF16),
                   dict(bias=BF16), dict(branch=1), dict(branch=7), dict(weight=F64, bias=F64),
                   dict(eps=-1.0), *SEEDS],
    "layer_norm_backward": [dict(d_y=(5, 24)), dict(d_y=(6, 20)), dict(d_total=(3, 24)),
                            dict(weight=(20,)), dict(weight=BF16), dict(stats=(11,)), dict(stats=F64),
                            dict(s=(7, 24)), dict(s=BF16), dict(s=F64), dict(param=1),
                            dict(branch=2, param=1), *SEEDS],
    "policy_loss": [dict(old=(5, 24)), dict(old=BF16), dict(ref=(6, 23)), dict(ref=F16),
                    dict(advantage=(5,)), dict(advantage=(6, 23)), dict(advantage=F16),
                    dict(mask=(6, 23)), dict(mask=torch.float32), dict(mask=torch.uint8),
                    dict(logp=F64), dict(reduction=4), dict(low=1.5)],
    "policy_loss_backward": [dict(old=(5, 24)), dict(ref=F16), dict(advantage=(5,)),
                             dict(mask=(6, 23)), dict(mask=torch.uint8), dict(grad=(1,)),
                             dict(grad=(6, 24)), dict(reduction=0), dict(share=(6,)),
                             dict(share=F64), dict(reduction=4)],
    "linear_cross_entropy": [dict(hidden=(6, 23)), dict(hidden=(2, 3, 24)), dict(hidden=F16),
                             dict(hidden=F64, weight=F64), dict(weight=(50, 20)), dict(weight=(24,)),
                             dict(weight=(0, 24)), dict(target=(5,)), dict(target=torch.int32),
                             dict(reduction=3)],
    "linear_cross_entropy_backward": [dict(hidden=(6, 23)), dict(hidden=F16), dict(weight=(50, 20)),
                                      dict(target=(5,)), dict(target=torch.int32), dict(grad=(6,)),
                                      dict(reduction=0), dict(reduction=3), dict(stats=(12,)),
                                      dict(stats=F16)],
}


def operands(name, change=()):
    out = []
    for key, value in CALLS[name].items():
        value = value(6, 24) if callable(value) else value
        if key in change:
            new = change[key]
            if isinstance(new, tuple):
                value = torch.ones(new, dtype=value.dtype, device=DEVICE)
            elif isinstance(new, torch.dtype):
                value = value.to(new)
            else:
                value = new.to(DEVICE) if isinstance(new, torch.Tensor) else new
        out.append(value)
    return out
