"""Layer norm of token rows on MI355X, differentiable.

The layer before the projection that MaxSim scores: every hidden state is
normalised over its d features. Extension of the reference API (no counterpart
in flash_maxsim 0.1.0, whose training starts at the token embeddings).

Rows are float16, bfloat16 or float32; sums, the mean and the deviation are
float32, and y and every gradient are rounded once. Weight and bias are of the
rows' type or float32, and so are their gradients, which are float32 sums in a
fixed order: the same inputs give the same bits.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .flash_maxsim import _check_devices, _device_guard

_CODES = {torch.float16: _lib.FMX_DTYPE_F16, torch.bfloat16: _lib.FMX_DTYPE_BF16, torch.float32: _lib.FMX_DTYPE_F32}


def _rows(t: torch.Tensor, d: int) -> torch.Tensor:
    """t as [M, d] rows with adjacent elements, in place where its strides allow."""
    t = t.resolve_neg().reshape(-1, d)
    return t if t.stride(1) == 1 or d == 1 else t.contiguous()


def _differentiated(*tensors) -> bool:
    """Whether autograd watches an operand (in forward mode too, which the Functions refuse)."""
    return torch.autograd.forward_ad._current_level >= 0 or (
        torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))


def _weight_type(x, weight, bias) -> torch.dtype:
    types = {t.dtype for t in (weight, bias) if t is not None}
    if not types:
        return x.dtype
    if len(types) > 1 or not types <= {x.dtype, torch.float32}:
        raise TypeError(f"weight and bias must both be {x.dtype} or both float32, got {sorted(map(str, types))}")
    return types.pop()


def _check(x, weight, bias) -> None:
    assert x.ndim >= 1 and x.size(-1) >= 1, "x must be [..., d] with d >= 1"
    for t in (weight, bias):
        assert t is None or tuple(t.shape) == (x.size(-1),), f"weight and bias must be [{x.size(-1)}]"
    if x.dtype not in _CODES:
        raise TypeError(f"x must be float16, bfloat16 or float32, got {x.dtype}")


def _forward(x, weight, bias, eps, save):
    """y, and with `save` the float32 mean and inverse deviation of each row."""
    d = x.size(-1)
    dev = _check_devices(x, weight, bias)
    wt = _weight_type(x, weight, bias)
    rows = _rows(x, d)
    weight = None if weight is None else weight.resolve_neg().contiguous()
    bias = None if bias is None else bias.resolve_neg().contiguous()
    M = rows.size(0)
    y = torch.empty(x.shape, device=dev, dtype=x.dtype)
    mean = torch.empty(M, device=dev, dtype=torch.float32) if save else None
    rstd = torch.empty(M, device=dev, dtype=torch.float32) if save else None
    with _device_guard(dev):
        rc = _lib.load().fmx_layer_norm(
            _CODES[x.dtype], rows.data_ptr(), rows.stride(0), _CODES[wt], _lib.ptr(weight), _lib.ptr(bias), M, d, eps,
            y.data_ptr(), _lib.ptr(mean), _lib.ptr(rstd), _lib.stream_of(x),
        )
    _lib.check(rc)
    return y, rows, weight, mean, rstd


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, rows, w, mean, rstd = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(rows, w, mean, rstd)
        ctx.wt = _weight_type(x, weight, bias)
        ctx.shape = x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rows, weight, mean, rstd = ctx.saved_tensors
        M, d = rows.shape
        # hooks on saved tensors may give them back in another layout
        rows, mean, rstd = _rows(rows, d), mean.contiguous(), rstd.contiguous()
        weight = None if weight is None else weight.resolve_neg().contiguous()
        dev = rows.device
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dys = _rows(dy, d)
        dx = torch.empty(ctx.shape, device=dev, dtype=rows.dtype) if need_x else None
        dw = torch.empty(d, device=dev, dtype=ctx.wt) if need_w else None
        db = torch.empty(d, device=dev, dtype=ctx.wt) if need_b else None
        lib = _lib.load()
        with _device_guard(dev):
            nbytes = lib.fmx_layer_norm_bwd_workspace_bytes(M, d) if need_w or need_b else 0
            ws = _lib.workspace(nbytes, dev)
            rc = lib.fmx_layer_norm_bwd(
                _CODES[rows.dtype], rows.data_ptr(), rows.stride(0), dys.data_ptr(), dys.stride(0), _CODES[ctx.wt],
                _lib.ptr(weight), mean.data_ptr(), rstd.data_ptr(), M, d, _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db),
                _lib.ptr(ws), nbytes, _lib.stream_of(rows),
            )
        _lib.check(rc)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    x is [..., d] with d from 1 to 65536, weight and bias [d] (ones and zeros
    where None); the variance is the biased one. The result has x's shape and
    type; differentiable in x, weight and bias.
    """
    out = _lib.native().layer_norm(x, weight, bias, eps)
    if out is not None:
        return out
    _check(x, weight, bias)
    if _differentiated(x, weight, bias):
        return _LayerNormFn.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]
