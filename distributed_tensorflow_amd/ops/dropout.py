"""Dropout whose mask is recomputed, never stored (``csrc/kernels/dropout.hip``).

``dropout(x, rate, seed, step)`` keeps element ``i`` (in row-major order) iff a 16-bit number drawn by the counter-based
generator Philox4x32-10 from ``(seed, step, i)`` is at least ``round(rate * 65536)``, and scales what it keeps by the
reciprocal of that keep probability.  The backward pass draws the same numbers again, so neither pass reads or writes a
mask, and results do not depend on launch shapes, streams or devices: CPU tensors get the same mask.  ``residual`` adds
the other branch of a residual block in the same pass.

``seed`` belongs to a layer (give each layer of a model its own; in a data-parallel run put the rank into it as well, or every
replica draws the same mask for its own rows), ``step`` to a call: an integer, or a one-element int64
tensor on x's device, whose value the kernel reads when it runs.  A captured graph that advances such a counter draws a
new mask in every replay; the backward pass uses the value that its forward pass saw.

Under activation checkpointing a forward pass runs twice.  ``FusedDropout`` then draws the first one's mask again (it knows
the call by a number from PyTorch's CPU generator, whose state ``torch.utils.checkpoint`` restores).  ``dropout`` is a
function: give the checkpointed part a ``step`` that has not moved on in between.

The reference has no dropout; the generator is the one of the truncated-normal initialiser (distributed.py:67-72).
"""
from __future__ import annotations

import ctypes as C
from collections import OrderedDict
from typing import Optional, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib, reference
from ._token import dtype_code, in_one_type, launch, same_device

_protos_done = False
REMEMBERED = 1024          # calls of a FusedDropout whose step is kept for a recomputation


def _kernels():
    global _protos_done
    lib = _lib.kernels()
    if not _protos_done:
        vp, u64 = C.c_void_p, C.c_uint64
        lib.dtf_dropout.restype = C.c_int
        lib.dtf_dropout.argtypes = [vp, vp, vp, C.c_int64, C.c_int, C.c_double, u64, u64, vp, vp, vp]
        _protos_done = True
    return lib


def dropout_apply(x: torch.Tensor, rate: float, seed: int, step: Union[int, torch.Tensor] = 0,
                  residual: Optional[torch.Tensor] = None, used: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[residual +] mask * x / keep`` without autograd; the same call on a gradient is the backward pass.  ``used``
    (one int64 on x's device) receives the step the mask was drawn with."""
    dt = dtype_code(x, "dropout: x")
    if not 0.0 <= rate <= 1.0:
        raise ValueError(f"dropout: rate must lie in [0, 1], got {rate}")
    if not 0 <= seed < 2 ** 64:
        raise ValueError("dropout: seed must be an unsigned 64-bit integer")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("dropout: residual must have x's shape and dtype")
    step_t = step if isinstance(step, torch.Tensor) else None
    for name, t in (("step", step_t), ("used", used)):
        if t is not None and (t.dtype != torch.int64 or t.numel() != 1):
            raise ValueError(f"dropout: {name} must be one int64")
    if step_t is None and not 0 <= step < 2 ** 63:
        raise ValueError("dropout: step must be a non-negative 63-bit integer")
    if used is not None and step_t is not None and used.data_ptr() == step_t.data_ptr():
        raise ValueError("dropout: used must not be the step counter itself")
    same_device("dropout", x, residual, step_t, used)
    if not x.is_cuda:
        value = int(step_t) if step_t is not None else int(step)
        if used is not None:
            used.fill_(value)
        return reference.dropout(x, rate, seed, value, residual)
    xc = x.contiguous()
    rc = residual.contiguous() if residual is not None else None
    y = x.new_empty(x.shape)
    launch("dropout", _kernels().dtf_dropout, x, xc.data_ptr(), _lib.ptr(rc), y.data_ptr(), xc.numel(), dt, rate, seed,
           0 if step_t is not None else step, _lib.ptr(step_t), _lib.ptr(used))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, rate, seed, step, used):
        if isinstance(step, torch.Tensor):                 # the counter may have moved on when backward() runs
            used = torch.empty(1, dtype=torch.int64, device=x.device) if used is None else used
        else:
            used = step
        y = dropout_apply(x, rate, seed, step, residual, used if used is not step else None)
        ctx.rate, ctx.seed, ctx.has_res = rate, seed, residual is not None
        ctx.step = used
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = dropout_apply(dy, ctx.rate, ctx.seed, ctx.step) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.has_res else None, None, None, None, None


def _dropout(x, rate, seed, step, residual, used=None):
    x, residual = in_one_type(x, residual)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, rate, seed, step, used)
    return dropout_apply(x, rate, seed, step, residual, used)


def dropout(x: torch.Tensor, rate: float, seed: int, step: Union[int, torch.Tensor] = 0,
            residual: Optional[torch.Tensor] = None, training: bool = True) -> torch.Tensor:
    """``[residual +] dropout(x)``; without ``training`` nothing is dropped.  Under autocast a residual of another type than
    ``x`` makes the result of the wider one."""
    if not training:
        return x if residual is None else x + residual
    return _dropout(x, rate, seed, step, residual)


class FusedDropout(nn.Module):
    """Dropout layer with its own seed and a step counter in device memory that every training call advances, in a
    captured graph as well.  The counter is a buffer: a restored checkpoint continues the mask sequence.

    A call inside a backward pass is a recomputation (activation checkpointing): it takes the step of the call it repeats and
    leaves the counter alone.  Each training call draws one number from PyTorch's CPU generator to be known by; where that
    number does not tell (``preserve_rng_state=False``, a generator seeded alike for several forward passes that wait
    for their backward pass, more than ``REMEMBERED`` calls in between) the recomputation raises."""

    def __init__(self, rate: float, seed: int):
        super().__init__()
        if not 0.0 <= rate <= 1.0:
            raise ValueError(f"FusedDropout: rate must lie in [0, 1], got {rate}")
        self.rate, self.seed = float(rate), int(seed)
        self.register_buffer("step", torch.zeros(1, dtype=torch.int64))
        self._steps = OrderedDict()               # number of the call -> [its step, recomputed already]; step None: several calls

    def __getstate__(self):
        return {**self.__dict__, "_steps": OrderedDict()}

    def _remember(self, call: int, used: torch.Tensor) -> None:
        known = self._steps.pop(call, None)
        # a call of the same number that still waits for its backward pass, or that never had one: which is meant?
        self._steps[call] = [used if known is None or known[1] else None, False]
        if len(self._steps) > REMEMBERED:
            self._steps.popitem(last=False)

    def forward(self, x, residual=None):              # noqa: D102
        if not self.training or self.rate == 0.0:
            return x if residual is None else x + residual
        call = int(torch.empty((), dtype=torch.int64, device="cpu").random_())
        if torch._C._current_graph_task_id() != -1:   # inside a backward pass
            known = self._steps.get(call)
            if known is None or known[0] is None:
                raise RuntimeError("FusedDropout: called inside a backward pass, but not as the recomputation of one known forward pass; "
                                   "activation checkpointing needs preserve_rng_state=True, or ops.dropout.dropout with a step of its own")
            known[1] = True
            return _dropout(x, self.rate, self.seed, known[0], residual)
        used = torch.empty_like(self.step)
        y = _dropout(x, self.rate, self.seed, self.step, residual, used)
        self._remember(call, used)
        with torch.no_grad():
            self.step.add_(1)
        return y

    def extra_repr(self) -> str:
        return f"rate={self.rate}, seed={self.seed}"
