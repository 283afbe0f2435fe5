"""Embedding lookup with scaling, and its gradient by sorted tokens (``csrc/kernels/embedding.hip``).

``embedding(ids, table, scale)`` is ``scale * table[ids]``.  The gradient of the table is a segmented sum over tokens
sorted by id: each row is written once, as the float32 sum of its tokens in the order of their positions times ``scale``,
rounded once, or as zeros.  No atomics: the same inputs give the same bits.

* ``ids``: int64 or int32 of any shape; ``table`` [V, D] float32 or bfloat16, its rows may be strided.
* An id outside the table raises on the CPU; on the GPU it gives a row of zeros and no gradient (what ``tf.gather``
  does on the two devices; raising would need a synchronisation).
* ``padding_idx``: tokens with this id give no gradient.

The reference looks up nothing but the rows of a batch; ``ops.gather_cast_transpose`` is that gather.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib, reference
from ._token import DTYPES, at_most, dtype_code, launch, rows_2d, same_device

_protos_done = False


def _kernels():
    global _protos_done
    lib = _lib.kernels()
    if not _protos_done:
        vp, i, i64, f = C.c_void_p, C.c_int, C.c_int64, C.c_float
        lib.dtf_embedding_fwd.restype = i
        lib.dtf_embedding_fwd.argtypes = [vp, i, vp, vp, i64, i64, i, i64, i, f, vp]
        lib.dtf_embedding_bwd_ws_bytes.restype = i64
        lib.dtf_embedding_bwd_ws_bytes.argtypes = [i64, i64, i]
        lib.dtf_embedding_bwd.restype = i
        lib.dtf_embedding_bwd.argtypes = [vp, i, vp, vp, vp, i64, i64, i64, i, i64, i, f, C.c_longlong, vp]
        _protos_done = True
    return lib


def _check_ids(ids):
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"embedding: ids must be int64 or int32, got {ids.dtype}")


def _padding(padding_idx, rows):
    if padding_idx is None:
        return -1                                          # never a valid id
    if not -rows <= padding_idx < rows:
        raise ValueError(f"embedding: padding_idx {padding_idx} lies outside the table of {rows} rows")
    return padding_idx % rows


def embedding_fwd(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[ids]`` of shape ``[*ids.shape, D]``, without autograd."""
    _check_ids(ids)
    if table.dim() != 2 or table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError("embedding: table must be [V, D]")
    dt = dtype_code(table, "embedding: table")
    at_most("embedding: width of the table", table.shape[1], 1 << 20)
    same_device("embedding", table, ids)
    if not table.is_cuda:
        return reference.embedding(ids, table, scale)
    t2, ldt = rows_2d(table, table.shape[1])
    ids = ids.contiguous()
    y = table.new_empty((*ids.shape, table.shape[1]))
    launch("embedding_fwd", _kernels().dtf_embedding_fwd, table, ids.data_ptr(), int(ids.dtype == torch.int64), t2.data_ptr(), y.data_ptr(),
           ids.numel(), table.shape[0], table.shape[1], ldt, dt, scale)
    return y


def embedding_bwd(dy: torch.Tensor, ids: torch.Tensor, rows: int, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """Gradient ``[rows, D]`` of the table, in ``dy``'s type, for the gradient ``dy`` ``[*ids.shape, D]`` of the lookup."""
    _check_ids(ids)
    if rows <= 0 or dy.dim() != ids.dim() + 1 or dy.shape[:-1] != ids.shape or dy.shape[-1] == 0:
        raise ValueError(f"embedding_bwd: dy must be [*ids.shape, D], got {tuple(dy.shape)} for ids {tuple(ids.shape)}")
    dt, cols = dtype_code(dy, "embedding_bwd: dy"), dy.shape[-1]
    at_most("embedding_bwd: width of the table", cols, 1 << 20)
    skip = _padding(padding_idx, rows)
    same_device("embedding_bwd", dy, ids)
    if not dy.is_cuda:
        return reference.embedding_bwd(dy, ids, rows, scale, padding_idx)
    lib = _kernels()
    d2, ldd = rows_2d(dy, cols)
    ids = ids.contiguous()
    n = ids.numel()
    need = lib.dtf_embedding_bwd_ws_bytes(n, rows, cols)
    if need < 0:
        raise ValueError(f"embedding_bwd: {n} tokens on a table of {rows} x {cols} are outside the kernels' range")
    out = torch.empty((rows, cols), dtype=dy.dtype, device=dy.device)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dy.device)
    launch("embedding_bwd", lib.dtf_embedding_bwd, dy, ids.data_ptr(), int(ids.dtype == torch.int64), d2.data_ptr(), out.data_ptr(), ws.data_ptr(),
           ws.numel(), n, rows, cols, ldd, dt, scale, skip)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.padding_idx = table.shape[0], scale, padding_idx
        return embedding_fwd(ids, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        return None, embedding_bwd(dy, ids, ctx.rows, ctx.scale, ctx.padding_idx), None, None


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * table[ids]``; tokens with id ``padding_idx`` give no gradient."""
    if padding_idx is not None and table.dim() == 2:
        _padding(padding_idx, table.shape[0])
    if torch.is_grad_enabled() and table.requires_grad:
        return _Embedding.apply(ids, table, scale, padding_idx)
    return embedding_fwd(ids, table, scale)


class ScaledEmbedding(nn.Embedding):
    """``nn.Embedding`` (same parameter and checkpoint name) whose output is multiplied by ``scale``."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0, padding_idx: Optional[int] = None, **kw):
        if kw.get("max_norm") is not None or kw.get("scale_grad_by_freq") or kw.get("sparse"):
            raise ValueError("ScaledEmbedding does not take max_norm, scale_grad_by_freq or sparse")
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, **kw)
        if self.weight.dtype not in DTYPES:
            raise ValueError("ScaledEmbedding: float32 or bfloat16")
        self.scale = float(scale)

    @classmethod
    def from_pretrained(cls, embeddings, freeze: bool = True, padding_idx: Optional[int] = None, scale: float = 1.0, **kw):
        """``nn.Embedding.from_pretrained`` with ``scale``."""
        m = super().from_pretrained(embeddings, freeze, padding_idx, **kw)
        m.scale = float(scale)
        return m

    def forward(self, ids):                           # noqa: D102
        return embedding(ids, self.weight, self.scale, self.padding_idx)
