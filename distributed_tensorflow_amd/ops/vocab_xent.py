"""Classifier + softmax cross entropy over a large vocabulary, without keeping the logits (``csrc/kernels/vocab_xent.hip``).

``vocab_xent(features, weight, labels, bias)`` is ``F.cross_entropy(F.linear(features, weight, bias), labels,
ignore_index=...)`` plus the hit count.  It stands beside ``classifier.linear_xent``, which stores the logits (and returns
them): here the forward pass reduces every logit to the row's statistics inside the product's epilogue, and the backward
pass recomputes the logits piece by piece of the vocabulary, so a call needs 8 bytes per 64 logits forward and a workspace
of about 1 GiB (or 16384 columns, whatever is more) backward, at any vocabulary size.

* types: float32 or bfloat16 features; a weight of the same type, or float32 under bfloat16 features (a bfloat16 copy is
  made piece by piece, its gradient is float32).  Logits, loss and statistics are float32.
* ``labels``: int64 class indices.  A row whose label is ``ignore_index`` has loss 0, gives no gradient and does not count,
  whatever its features hold (also NaN).
  A label outside the vocabulary raises on the CPU; on the GPU, where raising would need a synchronisation, its row's
  loss (and with it the total) is NaN and the row gives no gradient.
* ``reduction``: "mean" over the rows with a label (0 if there is none), "sum", or "none" (a loss per row).
* a class is taken out by the bias -inf.  Infinities in features and weight follow float32 arithmetic at every size (a product
  with -inf is -inf, 0 times an infinity is NaN, also in the features' gradient).
* the hit count is the number of rows with a label whose label is the first maximum of the row.

The reference's loss (distributed.py:81-87) is the ten-class case of this with logits kept; see ``classifier.py``.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib, reference
from ._token import DTYPES, at_most, dtype_code, launch, same_device

_protos_done = False
REDUCTIONS = ("mean", "sum", "none")


class _Args(C.Structure):
    """Mirror of ``DtfVocabXentArgs``."""
    _fields_ = [("X", C.c_void_p), ("W", C.c_void_p), ("bias", C.c_void_p), ("labels", C.c_void_p), ("lse", C.c_void_p),
                ("top", C.c_void_p), ("total", C.c_void_p), ("loss_rows", C.c_void_p), ("loss", C.c_void_p), ("counts", C.c_void_p), ("dloss", C.c_void_p),
                ("dX", C.c_void_p), ("dW", C.c_void_p), ("dbias", C.c_void_p), ("ws", C.c_void_p), ("ws_bytes", C.c_int64),
                ("ignore", C.c_longlong), ("ldx", C.c_int64), ("ldw", C.c_int64), ("V", C.c_int64), ("N", C.c_int),
                ("D", C.c_int), ("dtype", C.c_int), ("w_dtype", C.c_int), ("mean", C.c_int), ("dloss_rows", C.c_int)]


def _kernels():
    global _protos_done
    lib = _lib.kernels()
    if not _protos_done:
        pa = C.POINTER(_Args)
        lib.dtf_vocab_xent_ws_bytes.restype = C.c_int64
        lib.dtf_vocab_xent_ws_bytes.argtypes = [pa, C.c_int]
        for fn in (lib.dtf_vocab_xent_fwd, lib.dtf_vocab_xent_bwd):
            fn.restype = C.c_int
            fn.argtypes = [pa, C.c_void_p]
        _protos_done = True
    return lib


class VocabXentResult:
    """``loss`` (scalar; the sum for reduction "none"), ``loss_rows`` [N] and ``lse`` [N] in float32, ``hits`` and
    ``count`` (rows with a label) as int64 scalars on the device.  ``rows`` [4, N] holds what a row leaves: its loss, the
    logarithm of its sum of exponentials, its largest logit, and the sum of exponentials relative to that."""

    __slots__ = ("loss", "rows", "counts", "reduction", "ignore_index")

    def __init__(self, loss, rows, counts, reduction, ignore_index):
        self.loss, self.rows, self.counts = loss, rows, counts
        self.reduction, self.ignore_index = reduction, ignore_index

    @property
    def loss_rows(self) -> torch.Tensor:
        return self.rows[0]

    @property
    def lse(self) -> torch.Tensor:
        return self.rows[1]

    @property
    def hits(self) -> torch.Tensor:
        return self.counts[0]

    @property
    def count(self) -> torch.Tensor:
        return self.counts[1]


def _check(features, weight, labels, bias):
    if features.dim() != 2 or weight.dim() != 2 or features.shape[1] != weight.shape[1]:
        raise ValueError(f"vocab_xent: features [N, D] and weight [V, D], got {tuple(features.shape)} and {tuple(weight.shape)}")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError("vocab_xent: empty vocabulary or width")
    at_most("vocab_xent: rows", features.shape[0], 1 << 26)
    at_most("vocab_xent: width", features.shape[1], 1 << 20)
    code, wcode = dtype_code(features, "vocab_xent: features"), dtype_code(weight, "vocab_xent: weight")
    if wcode != code and wcode != 0:
        raise ValueError("vocab_xent: weight must have the features' dtype, or be float32")
    if labels.dim() != 1 or labels.shape[0] != features.shape[0] or labels.dtype != torch.int64:
        raise ValueError("vocab_xent: labels must be int64 [N]")
    if bias is not None and (tuple(bias.shape) != (weight.shape[0],) or bias.dtype not in DTYPES):
        raise ValueError("vocab_xent: bias must be float32 or bfloat16 [V]")
    same_device("vocab_xent", features, weight, labels, bias)
    return code, wcode


def _rows(t):
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if (t.shape[1] > 1 and t.stride(1) != 1) or ld < t.shape[1]:
        t, ld = t.contiguous(), t.shape[1]
    return t, ld


def _build(features, weight, labels, bias, rows, counts, ignore_index, mean):
    code, wcode = _check(features, weight, labels, bias)
    x, ldx = _rows(features)
    w, ldw = _rows(weight)
    b = None if bias is None else bias.detach().float().contiguous()
    labels = labels.contiguous()
    a = _Args()
    a.X, a.W, a.labels, a.counts = x.data_ptr(), w.data_ptr(), labels.data_ptr(), counts.data_ptr()
    at, step = rows.data_ptr(), 4 * rows.shape[1]
    a.loss_rows, a.lse, a.top, a.total = at, at + step, at + 2 * step, at + 3 * step
    a.bias = _lib.ptr(b)
    a.ignore, a.ldx, a.ldw, a.V, a.N, a.D = ignore_index, ldx, ldw, w.shape[0], x.shape[0], x.shape[1]
    a.dtype, a.w_dtype, a.mean = code, wcode, int(mean)
    return a, (x, w, b, labels)


def _workspace(a, backward, device):
    need = _kernels().dtf_vocab_xent_ws_bytes(C.byref(a), backward)
    if need < 0:
        raise ValueError(f"vocab_xent: [{a.N}, {a.D}] features with a vocabulary of {a.V} are outside the kernels' range "
                         "(an operand of 2 GiB or more: split the batch)")
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=device)
    a.ws, a.ws_bytes = ws.data_ptr(), ws.numel()
    return ws


def vocab_xent_fwd(features: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   ignore_index: int = -100, reduction: str = "mean") -> VocabXentResult:
    """Forward pass without autograd; see :class:`VocabXentResult`."""
    if reduction not in REDUCTIONS:
        raise ValueError(f"vocab_xent: reduction must be one of {REDUCTIONS}, got {reduction!r}")
    n, dev = features.shape[0], features.device
    if n == 0:
        _check(features, weight, labels, bias)
        return VocabXentResult(features.new_zeros((), dtype=torch.float32), features.new_zeros((4, 0), dtype=torch.float32),
                               labels.new_zeros(2), reduction, ignore_index)
    if not features.is_cuda:
        _check(features, weight, labels, bias)
        return VocabXentResult(*reference.vocab_xent(features, weight, labels, bias, ignore_index, reduction), reduction, ignore_index)
    rows = features.new_empty((4, n), dtype=torch.float32)
    loss = features.new_empty((), dtype=torch.float32)
    counts = features.new_empty(2, dtype=torch.int64)
    a, keep = _build(features, weight, labels, bias, rows, counts, ignore_index, reduction == "mean")
    a.loss = loss.data_ptr()
    ws = _workspace(a, 0, dev)
    launch("vocab_xent_fwd", _kernels().dtf_vocab_xent_fwd, features, C.byref(a))
    del keep, ws
    return VocabXentResult(loss, rows, counts, reduction, ignore_index)


def vocab_xent_bwd(fwd: VocabXentResult, features: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                   bias: Optional[torch.Tensor] = None, dloss: Optional[torch.Tensor] = None, want=(True, True, True)):
    """``(dfeatures, dweight, dbias)`` in the types of their tensors (dbias None without a bias).  ``dloss``: float32
    gradient of the loss, a scalar ("mean", "sum"; default 1) or one value a row ("none").  ``want``: which to compute."""
    want_x, want_w, want_b = want[0], want[1], want[2] and bias is not None
    n, dev = features.shape[0], features.device
    per_row = fwd.reduction == "none"
    if dloss is not None and (dloss.dtype != torch.float32 or dloss.numel() != (n if per_row else 1)):
        raise ValueError("vocab_xent_bwd: dloss must be float32, a scalar or (reduction \"none\") one value a row")
    same_device("vocab_xent_bwd", features, dloss, fwd.rows)
    if fwd.rows.shape[1] != n:
        raise ValueError("vocab_xent_bwd: the forward result belongs to another batch")
    if n == 0:
        _check(features, weight, labels, bias)
        return (torch.zeros_like(features) if want_x else None, weight.new_zeros(weight.shape) if want_w else None,
                bias.new_zeros(bias.shape) if want_b else None)
    if not features.is_cuda:
        _check(features, weight, labels, bias)
        d = reference.vocab_xent_bwd(features, weight, labels, bias, fwd.lse, fwd.counts, fwd.ignore_index, fwd.reduction, dloss)
        return d[0] if want_x else None, d[1] if want_w else None, d[2] if want_b else None
    a, keep = _build(features, weight, labels, bias, fwd.rows, fwd.counts, fwd.ignore_index, fwd.reduction == "mean")
    dx = torch.empty(features.shape, dtype=features.dtype, device=dev) if want_x else None
    dw = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if want_w else None
    db = torch.empty(weight.shape[0], dtype=torch.float32, device=dev) if want_b else None
    if not (want_x or want_w or want_b):
        return None, None, None
    g = None if dloss is None else dloss.contiguous()
    a.dloss, a.dloss_rows = _lib.ptr(g), int(per_row and g is not None)
    a.dX, a.dW, a.dbias = _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db)
    ws = _workspace(a, 1, dev)
    launch("vocab_xent_bwd", _kernels().dtf_vocab_xent_bwd, features, C.byref(a))
    del keep, ws, g
    return dx, dw, db.to(bias.dtype) if db is not None else None


class _VocabXent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, weight, labels, bias, ignore_index, reduction):
        r = vocab_xent_fwd(features, weight, labels, bias, ignore_index, reduction)
        ctx.save_for_backward(features, weight, labels, bias, r.rows, r.counts)
        ctx.reduction, ctx.ignore_index = reduction, ignore_index
        hits = r.counts[0].clone()
        ctx.mark_non_differentiable(hits)
        return (r.loss_rows.clone() if reduction == "none" else r.loss), hits       # what backward() reads stays its own

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _dhits):
        features, weight, labels, bias, rows, counts = ctx.saved_tensors
        fwd = VocabXentResult(None, rows, counts, ctx.reduction, ctx.ignore_index)
        need = (ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[3])
        dx, dw, db = vocab_xent_bwd(fwd, features, weight, labels, bias, dloss, need)
        return dx, dw, None, db, None, None


def vocab_xent(features: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, bias: Optional[torch.Tensor] = None,
               ignore_index: int = -100, reduction: str = "mean"):
    """``(loss, hits)``: cross entropy of ``features @ weight.T + bias`` against ``labels``, and the hit count."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (features, weight, bias)):
        return _VocabXent.apply(features, weight, labels, bias, ignore_index, reduction)
    r = vocab_xent_fwd(features, weight, labels, bias, ignore_index, reduction)
    return (r.loss_rows if reduction == "none" else r.loss), r.hits
