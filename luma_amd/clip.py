"""The global norm of many gradients, and clipping by it.

``get_total_norm``, ``clip_grad_norm_`` and ``clip_grads_with_norm_`` take the
arguments of ``torch.nn.utils``' functions of these names, which the
reference's benchmark calls between ``backward()`` and ``step()``
(benchmarks/bench_nanogpt.py)::

    loss.backward()
    norm = luma_amd.clip_grad_norm_(model.parameters(), 1.0)
    opt.step()

All gradients are read by one launch and, where they have to be clipped,
scaled in place by a second (luma_grad_clip in include/luma.h), with no host
synchronisation.  The norm is a float32 scalar on the gradients' device,
summed in float64, whatever the gradients' types.  Differences from torch:
float32, bfloat16 and float16 gradients on one ROCm GPU; p = 1, 2 or inf; a
parameter listed twice counts, and is clipped, once; the norm of bfloat16
gradients is not rounded to bfloat16.  ``make_fx`` and ``torch.jit.trace``
cannot record them (that raises); a HIP graph can capture them.

DTensor gradients (FSDP2) are normed by their local shards, the sums joined by
an all-reduce over the mesh dimensions that they are sharded over.
"""

from __future__ import annotations

import ctypes
import math
from typing import Iterable, List, Optional, Union

import numpy as np
import torch

from . import _lib as L

_GRAD_CODES = {torch.float32: L.GRAD_F32, torch.bfloat16: L.GRAD_BF16, torch.float16: L.GRAD_F16}
_NORMS = {2.0: L.NORM_L2, 1.0: L.NORM_L1, math.inf: L.NORM_INF}
_Tensors = Union[torch.Tensor, Iterable[torch.Tensor]]


def _norm_code(norm_type) -> int:
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"Invalid norm_type: {norm_type}. Expected 1, 2 or inf")
    return code


def check_max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"Invalid max_norm: {max_norm}")
    return max_norm


# Up to this many rows travel as launch arguments, a launch for each 160; more
# take a device table (a copy of 24 bytes per row, which a launch or two less
# does not pay for).  Under capture there is no table: the library takes up to
# 40,960 rows without one and refuses more.
NO_TABLE = 2 * L.GRADS_INLINE


class _Batch:
    """Dense gradients on one device as the rows of one call: a numpy array, or
    (host) a pinned tensor that holds them."""

    def __init__(self, rows: np.ndarray, device: torch.device, host=None, hold=None):
        self.rows = rows
        self.device = device
        self.host = host
        self.hold = hold      # keeps tensors alive that only the rows point to

    def zero(self) -> torch.Tensor:
        """The norm where there is no row."""
        return torch.zeros((), dtype=torch.float32, device=self.device)

    def args(self, norm: int, max_norm: float, total: Optional[torch.Tensor],
             power: Optional[torch.Tensor] = None) -> L.NormArgs:
        """The call's arguments, with a workspace (and, for a long list, a
        device copy of the rows) of their own."""
        partials = torch.empty(L.NORM_PARTIALS, dtype=torch.float64, device=self.device)
        table, n = None, len(self.rows)
        if n > NO_TABLE and not torch.cuda.is_current_stream_capturing():
            host = self.host
            if host is None:
                host = torch.from_numpy(self.rows.view(np.uint8)).pin_memory()
            # (on a stream of its own, beside what runs still, 20,000 tensors took
            # 644 us in place of 323: the wait between the streams costs more)
            table = host[:n * L.GRAD_DTYPE.itemsize].to(self.device, non_blocking=True)
        self.keep = (partials, table)
        return L.NormArgs(
            grads=self.rows.ctypes.data, table=None if table is None else table.data_ptr(), n=n,
            norm=norm, max_norm=max_norm, partials=partials.data_ptr(),
            total=None if total is None else total.data_ptr(),
            power=None if power is None else power.data_ptr())

    def call(self, name: str, args: L.NormArgs) -> None:
        lib = L.load()
        with torch.cuda.device(self.device):
            stream = torch.cuda.current_stream(self.device).cuda_stream
            L.check(getattr(lib, name)(ctypes.byref(args), stream), name)


def _check_not_recorded() -> None:
    """The calls below are no operators: a tracer would record the allocation of
    their outputs and not the kernels that fill them."""
    proxy = torch._C._TorchDispatchModeKey.PROXY
    if (torch._C._get_tracing_state() is not None
            or torch._C._get_dispatch_mode(proxy) is not None
            or torch._ops._get_dispatch_mode_pre_dispatch(proxy) is not None):
        raise RuntimeError("luma_amd: the gradients' norm and clipping cannot be recorded by make_fx "
                           "or torch.jit.trace (a HIP graph can capture them)")


def _host():
    return L.host_calls()


def _as_list(tensors: _Tensors) -> List[torch.Tensor]:
    if isinstance(tensors, torch.Tensor):
        return [tensors]
    return tensors if type(tensors) is list else list(tensors)


def _quick(tensors, of_grad: bool, apart: bool) -> Optional[_Batch]:
    """The rows by the host module, where every gradient can be taken as it is."""
    module = _host()
    if module is None:
        return None
    host, n = None, len(tensors)
    # (under capture the rows go as launch arguments, and nothing may be pinned)
    if (n > NO_TABLE and torch.cuda.is_available()
            and not torch.cuda.is_current_stream_capturing()):
        host = torch.empty(n * L.GRAD_DTYPE.itemsize, dtype=torch.uint8, pin_memory=True)
        rows = host.numpy().view(L.GRAD_DTYPE)
    else:
        rows = np.empty(n, dtype=L.GRAD_DTYPE)
    got = module.grad_rows(tensors, of_grad, apart, rows.ctypes.data)
    if got is None:
        return None
    # (no tensor at all has no device, and as in torch a norm on the host)
    device = torch.device("cpu") if got[1] < 0 else torch.device("cuda", got[1])
    return _Batch(rows[:got[0]], device, host)


def grad_rows(data, numel, dtype) -> np.ndarray:
    """The rows of gradients at these addresses, of these sizes (>= 1) and type codes."""
    rows = np.empty(len(numel), dtype=L.GRAD_DTYPE)
    rows["data"] = data
    rows["numel"] = numel
    rows["dtype"] = dtype
    tiles = (rows["numel"] + L.GRAD_TILE - 1) // L.GRAD_TILE
    if tiles.sum() >= 2**31:
        raise ValueError("luma_amd: too many gradient elements for one call")
    rows["first_tile"] = np.cumsum(tiles) - tiles
    return rows


def _rows(grads) -> np.ndarray:
    return grad_rows([g.data_ptr() for g in grads], [g.numel() for g in grads],
                     [_GRAD_CODES[g.dtype] for g in grads])


def _shard_dims(t) -> tuple:
    """The mesh dimensions over which a DTensor's elements are spread."""
    dims = []
    for d, place in enumerate(t.placements):
        if place.is_partial():
            raise ValueError("luma_amd: the norm of a DTensor with a Partial placement needs its "
                             "sum: redistribute it first")
        # (what a tensor-parallel weight's shards are cut into does not call itself a shard)
        if not place.is_replicate():
            dims.append(d)
    return tuple(dims)


def _check_device(g) -> None:
    if not g.is_cuda:
        raise RuntimeError(f"luma_amd: gradients must be on a ROCm GPU; got device {g.device}")


class _Slow:
    """Any gradients that torch knows: DTensors by their local shards, those
    that are not dense by a copy."""

    def __init__(self, grads, apart: bool):
        if apart:     # a gradient listed twice is one gradient
            grads = list({id(g): g for g in grads}.values())
        self.copies = []        # (a gradient that is not dense, its dense copy)
        self.sharded = {}       # (mesh, its dimensions) or None -> local gradients
        device = None
        for g in grads:
            key = None
            if hasattr(g, "_local_tensor") and hasattr(g, "device_mesh"):
                dims = _shard_dims(g)
                key = (g.device_mesh, dims) if dims else None
                g = g._local_tensor
            if g.is_sparse or g.layout != torch.strided:
                raise RuntimeError("luma_amd: sparse gradients are not supported")
            _check_device(g)
            if g.dtype not in _GRAD_CODES:
                raise ValueError(f"luma_amd: gradient dtype {g.dtype} is not "
                                 "float32/bfloat16/float16")
            device = device or g.device
            if g.device != device:
                raise RuntimeError("luma_amd: all gradients must be on one device "
                                   f"({device} vs {g.device})")
            if not _is_dense(g):
                dense = g.contiguous()
                self.copies.append((g, dense))
                g = dense
            self.sharded.setdefault(key, []).append(g)
        self.device = device
        self.batches = [(key, _Batch(_rows([g for g in gs if g.numel()]), device, hold=gs))
                        for key, gs in self.sharded.items()]
        if apart:
            _check_apart([g for gs in self.sharded.values() for g in gs if g.numel()])

    def norm(self, code: int) -> torch.Tensor:
        powers = []
        for key, batch in self.batches:
            power = torch.zeros((), dtype=torch.float64, device=self.device)
            if len(batch.rows):
                batch.call("luma_grad_norm", batch.args(code, 0.0, None, power))
            if key is not None:
                _join_shards(power, code, *key)
            powers.append(power)
        if code == L.NORM_INF:
            return torch.stack(powers).amax().float()
        power = torch.stack(powers).sum()
        return (power.sqrt() if code == L.NORM_L2 else power).float()

    def scale(self, max_norm: float, total: torch.Tensor) -> None:
        for _, batch in self.batches:
            if len(batch.rows):
                batch.call("luma_grad_scale", batch.args(L.NORM_L2, max_norm, total))
        torch.autograd.graph.increment_version(
            [g for gs in self.sharded.values() for g in gs if not g.is_inference()])
        for g, dense in self.copies:
            g.copy_(dense)


def _is_dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one run of memory, each once, in any order."""
    if t.is_neg() or t._is_zerotensor():
        return False
    span = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1),
                               key=lambda d: d[1]):
        if stride != span:
            return t.numel() == 0
        span *= size
    return True


def _check_apart(grads) -> None:
    spans = sorted((g.data_ptr(), g.data_ptr() + g.numel() * g.element_size()) for g in grads)
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError("luma_amd: gradients that share memory cannot be clipped in place")


def _join_shards(power: torch.Tensor, code: int, mesh, dims) -> None:
    """The power over all shards: summed (the largest one for inf) along each
    of the mesh's dimensions."""
    import torch.distributed as dist

    op = dist.ReduceOp.SUM
    if code == L.NORM_INF:
        # (by its bits, as the kernels keep it, NaN above infinity: a maximum of
        # floats may lose a NaN, and not on every rank)
        op, power = dist.ReduceOp.MAX, power.view(torch.int64)
    for d in dims:
        dist.all_reduce(power, op=op, group=mesh.get_group(d))


def _grads(params) -> List[torch.Tensor]:
    return [p.grad for p in params if p.grad is not None]


def _check_finite(total: torch.Tensor, norm_type) -> None:
    if not torch.isfinite(total):
        raise RuntimeError(
            f"The total norm of order {float(norm_type)} for gradients from `parameters` is "
            "non-finite, so it cannot be clipped. To disable this error and scale the gradients "
            "by the non-finite norm anyway, set `error_if_nonfinite=False`")


def sharded_norm(grads) -> Optional[torch.Tensor]:
    """The 2-norm of gradients some of which are spread over several GPUs; None
    where none is."""
    if not any(hasattr(g, "_local_tensor") and _shard_dims(g) for g in grads):
        return None
    return _Slow(grads, False).norm(L.NORM_L2)


def _quick_norm(tensors, clip: bool, code: int, max_norm: float) -> Optional[torch.Tensor]:
    """The whole call by the host module, for a list without a device table."""
    host = _host()
    return None if host is None else host.grad_norm(tensors, clip, code, max_norm, NO_TABLE)


@torch.compiler.disable
def get_total_norm(tensors: _Tensors, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                   foreach: Optional[bool] = None) -> torch.Tensor:
    """The norm of all elements of all tensors together (``norm_type`` 1, 2 or
    inf), as a float32 scalar on their device.  ``foreach`` is accepted for
    torch's signature and selects nothing."""
    _check_not_recorded()
    code = _norm_code(norm_type)
    tensors = _as_list(tensors)
    total = _quick_norm(tensors, False, code, 0.0)
    if total is None:
        total = _total_norm(tensors, code)
    if error_if_nonfinite:
        _check_finite(total, norm_type)
    return total


@torch.no_grad()
def _total_norm(tensors, code: int) -> torch.Tensor:
    if not tensors:
        return torch.tensor(0.0)
    batch = _quick(tensors, False, False)
    if batch is None:
        return _Slow(tensors, False).norm(code)
    if not len(batch.rows):
        return batch.zero()
    total = torch.empty((), dtype=torch.float32, device=batch.device)
    batch.call("luma_grad_norm", batch.args(code, 0.0, total))
    return total


@torch.compiler.disable
def clip_grad_norm_(parameters: _Tensors, max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False,
                    foreach: Optional[bool] = None) -> torch.Tensor:
    """Scales the parameters' gradients in place by
    ``min(1, max_norm / (norm + 1e-6))``, ``norm`` being the norm of all of
    them together, which is returned (a float32 scalar on their device).  A norm
    that is not finite scales by 0 or NaN, as in torch, unless
    ``error_if_nonfinite``, which waits for the norm and raises."""
    _check_not_recorded()
    code = _norm_code(norm_type)
    max_norm = check_max_norm(max_norm)
    parameters = _as_list(parameters)
    if not error_if_nonfinite:
        total = _quick_norm(parameters, True, code, max_norm)
        if total is not None:
            return total
    return _clip(parameters, max_norm, norm_type, code, error_if_nonfinite)


@torch.no_grad()
def _clip(parameters, max_norm: float, norm_type, code: int,
          error_if_nonfinite: bool) -> torch.Tensor:
    batch = None if error_if_nonfinite else _quick(parameters, True, True)
    if batch is not None:
        if not len(batch.rows):
            return batch.zero()
        total = torch.empty((), dtype=torch.float32, device=batch.device)
        batch.call("luma_grad_clip", batch.args(code, max_norm, total))
        return total
    grads = _grads(parameters)
    if not grads:
        return torch.tensor(0.0)
    slow = _Slow(grads, True)
    total = slow.norm(code)
    if error_if_nonfinite:
        _check_finite(total, norm_type)
    slow.scale(max_norm, total)
    return total


@torch.compiler.disable
@torch.no_grad()
def clip_grads_with_norm_(parameters: _Tensors, max_norm: float, total_norm: torch.Tensor,
                          foreach: Optional[bool] = None) -> None:
    """The scaling of ``clip_grad_norm_`` by a norm that is known already (a
    one-element tensor, e.g. ``get_total_norm``'s)."""
    _check_not_recorded()
    max_norm = check_max_norm(max_norm)
    parameters = _as_list(parameters)
    if not isinstance(total_norm, torch.Tensor) or total_norm.numel() != 1:
        raise ValueError("clip_grads_with_norm_: total_norm must be a one-element tensor")
    batch = _quick(parameters, True, True)
    if batch is not None:
        if len(batch.rows):
            total = total_norm.to(device=batch.device, dtype=torch.float32)
            batch.call("luma_grad_scale", batch.args(L.NORM_L2, max_norm, total))
        return
    grads = _grads(parameters)
    if grads:
        slow = _Slow(grads, True)
        slow.scale(max_norm, total_norm.to(device=slow.device, dtype=torch.float32))
