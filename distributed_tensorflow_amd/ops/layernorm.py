"""Layer normalisation over the last axis on the framework's kernels (``csrc/kernels/layernorm.hip``).

``layer_norm(x, weight, bias, eps)`` is ``F.layer_norm`` over the last axis; with ``residual`` it normalises the sum
``h = x + residual`` and returns ``(y, h)``, the two tensors a residual block hands on, in one pass over memory.  Forward
is one launch, backward two (the second adds the weight gradient's partial sums in a fixed order, so results are
reproducible bit for bit).  ``layer_norm_fwd`` / ``layer_norm_bwd`` are the same kernels without autograd.

Types: float32 and bfloat16 activations of any width, float32 or bfloat16 parameters; sums and statistics are float32
and results are rounded once.  ``h`` is rounded to the activations' type first and normalised as stored, which is what
the backward pass reads.  Rows may be strided; other layouts are copied.  CPU tensors take the plain statement
(``reference.layer_norm``).

The reference has no normalisation layer (distributed.py:78-81 is the whole network); like ``ops/batchnorm.py`` this is
a building block for module programs.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib, reference
from ._token import at_most, dtype_code, in_one_type, launch, rows_2d, same_device

_protos_done = False


def _kernels():
    global _protos_done
    lib = _lib.kernels()
    if not _protos_done:
        vp, i, i64, f = C.c_void_p, C.c_int, C.c_int64, C.c_float
        lib.dtf_layernorm_fwd.restype = i
        lib.dtf_layernorm_fwd.argtypes = [vp] * 8 + [i64, i, i64, i64, i, i, f, vp]
        lib.dtf_layernorm_bwd.restype = i
        lib.dtf_layernorm_bwd.argtypes = [vp] * 10 + [i64, i, i64, i64, i64, i, i, vp]
        lib.dtf_layernorm_bwd_ws_floats.restype = i64
        lib.dtf_layernorm_bwd_ws_floats.argtypes = [i64, i]
        _protos_done = True
    return lib


class LayerNormResult:
    """``y``, the normalised tensor ``h`` (``x``, or ``x + residual`` as stored) and its float32 row statistics ``stats``
    [2, rows] = (mean, 1 / standard deviation), which the backward pass reads."""

    __slots__ = ("y", "h", "stats")

    def __init__(self, y, h, stats):
        self.y, self.h, self.stats = y, h, stats

    @property
    def mean(self) -> torch.Tensor:
        return self.stats[0]

    @property
    def rstd(self) -> torch.Tensor:
        return self.stats[1]


def _param_code(what, x, weight, bias):
    cols = x.shape[-1]
    code = 0
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.dim() != 1 or p.shape[0] != cols or not p.is_contiguous():
            raise ValueError(f"{what}: {name} must be a contiguous [{cols}] tensor, got {tuple(p.shape)}")
        code = dtype_code(p, f"{what}: {name}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"{what}: weight and bias must have one dtype")
    return code


def layer_norm_fwd(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                   eps: float = 1e-5, residual: Optional[torch.Tensor] = None) -> LayerNormResult:
    """Forward pass; see :class:`LayerNormResult`."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("layer_norm: x needs a last axis of at least one element")
    dt, cols = dtype_code(x, "layer_norm: x"), x.shape[-1]
    at_most("layer_norm: last axis", cols, 1 << 30)
    wcode = _param_code("layer_norm", x, weight, bias)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("layer_norm: residual must have x's shape and dtype")
    if not eps >= 0.0:
        raise ValueError("layer_norm: eps must not be negative")
    same_device("layer_norm", x, weight, bias, residual)
    if not x.is_cuda:
        y, h, mean, rstd = reference.layer_norm(x, weight, bias, eps, residual)
        return LayerNormResult(y, h, torch.stack((mean, rstd)))
    x2, ldx = rows_2d(x, cols)
    r2, ldr = rows_2d(residual, cols) if residual is not None else (None, 0)
    rows = x.numel() // cols
    y = x.new_empty(x.shape)
    h = x.new_empty(x.shape) if r2 is not None else None
    stats = x.new_empty((2, rows), dtype=torch.float32)
    mean = stats.data_ptr()
    launch("layer_norm_fwd", _kernels().dtf_layernorm_fwd, x, x2.data_ptr(), _lib.ptr(r2), _lib.ptr(weight), _lib.ptr(bias),
           y.data_ptr(), _lib.ptr(h), mean, mean + 4 * rows, rows, cols, ldx, ldr, dt, wcode, eps)
    return LayerNormResult(y, x2 if h is None else h, stats)


def layer_norm_bwd(dy: torch.Tensor, fwd: LayerNormResult, weight: Optional[torch.Tensor] = None,
                   dh: Optional[torch.Tensor] = None, want_wgrad: bool = True):
    """``(dx, dweight, dbias)`` for the gradient ``dy`` of ``fwd.y``.  With a residual the same ``dx`` is the gradient of
    both addends, and ``dh`` is what the other users of ``fwd.h`` contribute to it.  The parameters' gradients have the
    weight's type (float32 without one) and are None where ``want_wgrad`` is false."""
    h = fwd.h
    cols = h.shape[-1]
    dt = dtype_code(h, "layer_norm_bwd: h")
    at_most("layer_norm_bwd: last axis", cols, 1 << 30)
    wcode = _param_code("layer_norm_bwd", h, weight, None)
    for name, t in (("dy", dy), ("dh", dh)):
        if t is not None and (t.numel() != h.numel() or t.shape[-1] != cols or t.dtype != h.dtype):
            raise ValueError(f"layer_norm_bwd: {name} must have the shape and dtype of the normalised tensor")
    same_device("layer_norm_bwd", h, dy, weight, dh)
    wdtype = torch.float32 if weight is None else weight.dtype
    if not h.is_cuda:
        dx, dw, db = reference.layer_norm_bwd(dy, h, fwd.mean, fwd.rstd, weight, dh)
        return (dx, dw.to(wdtype), db.to(wdtype)) if want_wgrad else (dx, None, None)
    lib = _kernels()
    h2, ldh = rows_2d(h, cols)
    dy2, lddy = rows_2d(dy, cols)
    dh2, lddh = rows_2d(dh, cols) if dh is not None else (None, 0)
    rows, mean = h.numel() // cols, fwd.stats.data_ptr()
    dx = h.new_empty(dy.shape)
    dw = db = part = None
    if want_wgrad:
        grads = h.new_empty((2, cols), dtype=wdtype)
        dw, db = grads[0], grads[1]
        part = h.new_empty(lib.dtf_layernorm_bwd_ws_floats(rows, cols), dtype=torch.float32)
    launch("layer_norm_bwd", lib.dtf_layernorm_bwd, h, dy2.data_ptr(), h2.data_ptr(), _lib.ptr(dh2), _lib.ptr(weight),
           mean, mean + 4 * rows, dx.data_ptr(), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(part), rows, cols,
           lddy, ldh, lddh, dt, wcode)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        r = layer_norm_fwd(x, weight, bias, eps, residual)
        ctx.save_for_backward(r.h, r.stats, weight)
        ctx.shape, ctx.has_res, ctx.has_bias = x.shape, residual is not None, bias is not None
        ctx.bdtype = bias.dtype if bias is not None else None
        ctx.set_materialize_grads(False)
        return (r.y, r.h) if residual is not None else r.y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, stats, weight = ctx.saved_tensors
        dw = db = None
        if dy is None:
            dx = dh                                        # only the sum itself was used
        else:
            need = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
            dx, dw, db = layer_norm_bwd(dy, LayerNormResult(None, h, stats), weight, dh, want_wgrad=need)
            dx = dx.view(ctx.shape)
        return (dx, dx if ctx.has_res else None, dw if weight is not None else None,
                db.to(ctx.bdtype) if db is not None and ctx.has_bias else None, None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, residual: Optional[torch.Tensor] = None):
    """``y``, or ``(y, h)`` with a residual: layer normalisation of ``x [+ residual]`` over the last axis.  Under autocast a
    residual of another type than ``x`` makes both results of the wider one."""
    x, residual = in_one_type(x, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, bias)):
        return _LayerNorm.apply(x, residual, weight, bias, eps)
    r = layer_norm_fwd(x, weight, bias, eps, residual)
    return (r.y, r.h) if residual is not None else r.y


class FusedLayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last axis (same parameters and checkpoint names) with an optional residual addition:
    ``forward(x)`` is ``y``, ``forward(x, residual)`` is ``(y, x + residual)``."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, **kw):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, **kw)
        if len(self.normalized_shape) != 1:
            raise ValueError("FusedLayerNorm normalises the last axis only")

    def forward(self, x, residual=None):              # noqa: D102
        if x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"FusedLayerNorm: last axis is {x.shape[-1]}, expected {self.normalized_shape[0]}")
        return layer_norm(x, self.weight, self.bias, self.eps, residual)
