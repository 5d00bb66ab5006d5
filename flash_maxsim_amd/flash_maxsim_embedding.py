"""Embedding lookup with scaling on MI355X, differentiable.

The first layer of a token encoder: ids become hidden states. Extension of the
reference API (no counterpart in flash_maxsim 0.1.0, whose training starts at the
token embeddings).

The table is float16, bfloat16 or float32; a row is scaled in float32 and rounded once.
The table's gradient sorts the tokens by id and sums the rows of each in float32 in a
fixed order, rounded once: the same inputs give the same bits, whatever ids repeat.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .flash_maxsim import _check_devices, _device_guard
from .flash_maxsim_norm import _CODES, _differentiated, _rows

MAX_TOKENS, MAX_ROWS = 1 << 26, 1 << 28


def _check(ids, weight, scale, padding_idx) -> None:
    assert weight.ndim == 2 and weight.size(0) >= 1 and weight.size(1) >= 1, "weight must be [V, d] with V and d >= 1"
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"ids must be int64 or int32, got {ids.dtype}")
    if weight.dtype not in _CODES:
        raise TypeError(f"weight must be float16, bfloat16 or float32, got {weight.dtype}")
    if not math.isfinite(scale):
        raise ValueError(f"scale={scale} must be finite")
    if padding_idx is not None and not 0 <= padding_idx < weight.size(0):
        raise ValueError(f"padding_idx={padding_idx} must be a row of the table, 0 .. {weight.size(0) - 1}")


def _forward(ids, weight, scale):
    """y, and the ids as the kernels read them."""
    dev = _check_devices(weight, ids)
    ids = ids.resolve_neg().contiguous()
    rows = _rows(weight, weight.size(1))
    V, d = weight.shape
    y = torch.empty(*ids.shape, d, device=dev, dtype=weight.dtype)
    with _device_guard(dev):
        rc = _lib.load().fmx_embedding(_CODES[weight.dtype], ids.data_ptr(), 64 if ids.dtype == torch.int64 else 32,
                                       rows.data_ptr(), rows.stride(0), scale, ids.numel(), V, d, y.data_ptr(),
                                       _lib.stream_of(weight))
    _lib.check(rc)
    return y, ids


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding):
        y, ids = _forward(ids, weight, scale)
        ctx.save_for_backward(ids)
        ctx.shape, ctx.how = weight.shape, (scale, padding)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if not ctx.needs_input_grad[1]:
            return None, None, None, None
        _lib.native().refuse_capture(ctx)
        (ids,) = ctx.saved_tensors
        ids = ids.resolve_neg().contiguous()
        V, d = ctx.shape
        scale, padding = ctx.how
        T, dev = ids.numel(), dy.device
        dw = torch.empty(V, d, device=dev, dtype=dy.dtype)
        dys = _rows(dy, d)
        lib, code = _lib.load(), _CODES[dy.dtype]
        with _device_guard(dev):
            nbytes = lib.fmx_embedding_bwd_workspace_bytes(code, T, V, d)
            ws = _lib.workspace(nbytes, dev)
            rc = lib.fmx_embedding_bwd(code, ids.data_ptr(), 64 if ids.dtype == torch.int64 else 32, dys.data_ptr(),
                                       dys.stride(0), scale, padding, T, V, d, dw.data_ptr(), _lib.ptr(ws), nbytes,
                                       _lib.stream_of(dys))
        _lib.check(rc)
        return None, dw, None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """scale * weight[ids]: [..., d] in weight's type.

    ids is [...] of int64 or int32, weight [V, d]. Ids outside 0 .. V - 1 give
    rows of NaN (a launch cannot raise) and no gradient. Differentiable in
    weight, with a dense gradient; tokens of padding_idx add nothing to it.
    """
    if math.isfinite(scale) and (padding_idx is None or (type(padding_idx) is int and padding_idx >= 0)):
        out = _lib.native().embedding(ids, weight, float(scale), -1 if padding_idx is None else padding_idx)
        if out is not None:
            return out
    _check(ids, weight, scale, padding_idx)
    scale, padding = float(scale), -1 if padding_idx is None else int(padding_idx)
    if _differentiated(weight):
        return _EmbeddingFn.apply(ids, weight, scale, padding)
    return _forward(ids, weight, scale)[0]
