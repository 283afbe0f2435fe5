"""What the token-model operators (``layernorm``, ``dropout``, ``embedding``, ``vocab_xent``) share: operand checks and
the launch on a tensor's own device and stream.

Workspaces come from PyTorch's allocator call by call: each belongs to the stream the call runs on, and to the graph
that captured it, so neither two streams nor two graphs ever share one.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1}       # element type codes of the C entry points


def dtype_code(t: torch.Tensor, what: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: expected float32 or bfloat16, got {t.dtype}")
    return code


def at_most(what: str, n: int, most: int) -> None:
    """Sizes that the C entry points take as 32-bit numbers: refused here, before they could wrap."""
    if n > most:
        raise ValueError(f"{what}: {n} is beyond the kernels' range of {most}")


def same_device(what: str, first: torch.Tensor, *others) -> None:
    """Operands of one device; on a GPU none with a forward-mode tangent, which a kernel would drop without a word."""
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on different devices: {dev} vs {t.device}")
    if forward_ad._current_level >= 0 and dev.type != "cpu":
        refuse_tangents(what, first, *others)


def refuse_tangents(what: str, *tensors) -> None:
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what}: no forward-mode derivative on the GPU (CPU tensors have one)")


def in_one_type(x: torch.Tensor, residual):
    """Under autocast a branch comes in autocast's type and the residual stream in float32: both in the wider type, as in
    ``x + residual``."""
    if residual is not None and residual.dtype != x.dtype and torch.is_autocast_enabled(x.device.type):
        wide = torch.promote_types(x.dtype, residual.dtype)
        return x.to(wide), residual.to(wide)
    return x, residual


def rows_2d(t: torch.Tensor, cols: int):
    """``t`` (last axis of ``cols`` elements) as rows and the distance between them; a copy only where no such view exists."""
    if t.is_contiguous():
        return t, cols
    r = t.reshape(-1, cols)
    ld = r.stride(0) if r.shape[0] > 1 else cols
    if (cols > 1 and r.stride(1) != 1) or ld < cols:
        r, ld = r.contiguous(), cols
    return r, ld


def launch(what: str, fn, t: torch.Tensor, *args) -> None:
    """``fn(*args, stream)`` on the current stream of ``t``'s device, whatever the current device is."""
    index = t.device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, what)
