"""Linear layer with bias, activation and residual in its epilogue, on MI355X.

What turns an encoder's hidden states into the token embeddings that MaxSim
scores: y = act(x W^T + bias) + residual in one pass, and its backward. Extension
of the reference API (no counterpart in flash_maxsim 0.1.0, whose training starts
at the token embeddings).

Operands are all float16 or all bfloat16; products run on MFMA with float32 sums,
and y is rounded once. The backward rounds dz = dy act'(z) to the operands' type,
as MFMA takes it; the slopes act'(z) are kept between the passes in 16 bits (only
with an activation), whose steps get finer towards zero: at most 2^-14 (bfloat16:
2^-13) of the slope down to 0.28 (0.07), and slopes down to 2^-30 (2^-60) are not
lost. Bias gradients sum the unrounded dz. Sums have a fixed order: the same
inputs give the same bits.

x and weight are read in place when their rows are 16-byte aligned and K is a
multiple of 8; other layouts are copied once per call with K zero-padded to a
multiple of 8.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib
from .flash_maxsim import _abi_ready, _check_devices, _device_guard, _own_strides
from .flash_maxsim_norm import _differentiated, _rows

ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _operand(t: torch.Tensor) -> torch.Tensor:
    """[rows, K] as the kernels read it: t itself, or a copy with K zero-padded to a multiple of 8."""
    t = t.resolve_neg()
    K = t.shape[1]
    if K % 8 == 0 and _abi_ready(t, None) and t.stride(0) < 1 << 22:
        return t
    t = F.pad(t, (0, -K % 8)) if K % 8 else _own_strides(t.contiguous())
    return t.clone() if t.data_ptr() % 16 else t


def _check(x, weight, bias, activation, residual) -> None:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation={activation!r} must be one of {list(ACTIVATIONS)}")
    assert x.ndim >= 1 and weight.ndim == 2 and x.size(-1) == weight.size(1), "x must be [..., K] and weight [N, K]"
    N, K = weight.shape
    assert N >= 1 and K >= 1, "weight must have rows and columns"
    assert bias is None or tuple(bias.shape) == (N,), f"bias must be [{N}]"
    assert residual is None or tuple(residual.shape) == (*x.shape[:-1], N), "residual must be [..., N]"
    types = {t.dtype for t in (x, weight, bias, residual) if t is not None}
    if types not in ({torch.float16}, {torch.bfloat16}):
        raise TypeError(f"x, weight, bias and residual must all be float16 or all bfloat16, got {sorted(map(str, types))}")


def _forward(x, weight, bias, act, residual, save):
    """y, the operands as the kernels read them, and with `save` and an activation its slopes."""
    N, K = weight.shape
    dev = _check_devices(x, weight, bias, residual)
    xk, wk = _operand(_rows(x, K)), _operand(weight)
    res = None if residual is None else _rows(residual, N)
    bias = None if bias is None else bias.resolve_neg().contiguous()
    M = xk.size(0)
    y = torch.empty(*x.shape[:-1], N, device=dev, dtype=x.dtype)
    slope = torch.empty(M, N, device=dev, dtype=torch.int16) if save and act else None
    lib = _lib.load()
    with _device_guard(dev):
        nbytes = lib.fmx_linear_workspace_bytes(M, N, K)
        ws = _lib.workspace(nbytes, dev)
        rc = lib.fmx_linear(
            _lib.dtype_code(xk), xk.data_ptr(), xk.stride(0), wk.data_ptr(), wk.stride(0), _lib.ptr(bias),
            _lib.ptr(res), 0 if res is None else res.stride(0), act, M, N, K, y.data_ptr(), _lib.ptr(slope),
            _lib.ptr(ws), nbytes, _lib.stream_of(x),
        )
    _lib.check(rc)
    return y, xk, wk, slope


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act, residual):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        y, xk, wk, slope = _forward(x, weight, bias, act, residual, need_x or need_w or need_b)
        # dx reads w, dw reads x: an operand that no wanted gradient needs is free to go or to change
        ctx.save_for_backward(xk if need_w else None, wk if need_x else None, slope)
        ctx.act, ctx.shape, ctx.sizes = act, x.shape, (xk.size(0), *weight.shape)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _lib.native().refuse_capture(ctx)
        xk, wk, slope = ctx.saved_tensors
        # hooks on saved tensors may give them back in another layout
        xk, wk = (None if t is None else _operand(t) for t in (xk, wk))
        slope = None if slope is None else slope.contiguous()
        (M, N, K), dev = ctx.sizes, dy.device
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = torch.empty(ctx.shape, device=dev, dtype=dy.dtype) if need_x else None
        dw = torch.empty(N, K, device=dev, dtype=dy.dtype) if need_w else None
        db = torch.empty(N, device=dev, dtype=dy.dtype) if need_b else None
        if need_x or need_w or need_b:
            dys = _rows(dy, N)
            lib = _lib.load()
            with _device_guard(dev):
                nbytes = lib.fmx_linear_bwd_workspace_bytes(M, N, K)
                ws = _lib.workspace(nbytes, dev)
                rc = lib.fmx_linear_bwd(
                    _lib.dtype_code(dy), _lib.ptr(xk), 0 if xk is None else xk.stride(0), _lib.ptr(wk),
                    0 if wk is None else wk.stride(0), dys.data_ptr(), dys.stride(0), _lib.ptr(slope), ctx.act, M, N, K,
                    _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws), nbytes, _lib.stream_of(dys),
                )
            _lib.check(rc)
        return dx, dw, db, None, dy if ctx.needs_input_grad[4] else None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """act(x W^T + bias) + residual: [..., N] in x's type.

    x is [..., K], weight [N, K], bias [N], residual [..., N]; activation is
    None, "relu", "gelu" (by the normal distribution function), "gelu_tanh" (its
    tanh form) or "silu". Differentiable in x, weight, bias and residual.
    """
    out = _lib.native().linear(x, weight, bias, ACTIVATIONS.get(activation, -1), residual)
    if out is not None:
        return out
    _check(x, weight, bias, activation, residual)
    act = ACTIVATIONS[activation]
    if _differentiated(x, weight, bias, residual):
        return _LinearFn.apply(x, weight, bias, act, residual)
    return _forward(x, weight, bias, act, residual, False)[0]
