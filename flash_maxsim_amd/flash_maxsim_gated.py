"""Gated linear layer on MI355X: both projections, the activation and their product in one kernel.

The first half of an encoder block's gated feed-forward layer: y = act(x Wg^T + bg) * (x Wu^T + bu);
`linear`, with the block's residual, is the second. Extension of the reference API
(no counterpart in flash_maxsim 0.1.0, whose training starts at the token embeddings).

Operands are all float16 or all bfloat16; products run on MFMA with float32 sums,
and y is rounded once: neither product reaches memory. The backward rounds
dg = dy u act'(g) and du = dy act(g) to the operands' type, as MFMA takes them; the
factors u act'(g) and act(g) are kept between the passes in codes of more bits than
the operands have (bfloat16: 16, fp16: 24; off by 2^-10 and 2^-16 of the factor at
most; bfloat16 outside 2^-16 .. 2^16 by 2^-8, and beyond 2^79 a factor is NaN). Bias gradients sum the unrounded dg and du. Sums have
a fixed order: the same inputs give the same bits.

x and the weights are read in place when their rows are 16-byte aligned and K is a
multiple of 8 (halves of one fused weight are such views); other layouts are copied
once per call with K zero-padded to a multiple of 8.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .flash_maxsim import _check_devices, _device_guard
from .flash_maxsim_linear import ACTIVATIONS, _operand
from .flash_maxsim_norm import _differentiated, _rows


def _planes(dtype: torch.dtype) -> int:
    return 2 if dtype == torch.bfloat16 else 3


def _check(x, weight_gate, weight_up, bias_gate, bias_up, activation) -> None:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation={activation!r} must be one of {list(ACTIVATIONS)}")
    assert x.ndim >= 1 and weight_gate.ndim == 2 and weight_gate.shape == weight_up.shape, \
        "x must be [..., K], weight_gate and weight_up [N, K]"
    N, K = weight_gate.shape
    assert x.size(-1) == K, "x must be [..., K], weight_gate and weight_up [N, K]"
    assert N >= 1 and K >= 1, "the weights must have rows and columns"
    for b in (bias_gate, bias_up):
        assert b is None or tuple(b.shape) == (N,), f"bias_gate and bias_up must be [{N}]"
    types = {t.dtype for t in (x, weight_gate, weight_up, bias_gate, bias_up) if t is not None}
    if types not in ({torch.float16}, {torch.bfloat16}):
        raise TypeError(f"x, weights and biases must all be float16 or all bfloat16, got {sorted(map(str, types))}")


def _forward(x, weight_gate, weight_up, bias_gate, bias_up, act, save):
    """y, the operands as the kernels read them, and with `save` the backward's factors."""
    N, K = weight_gate.shape
    dev = _check_devices(x, weight_gate, weight_up, bias_gate, bias_up)
    xk, wg, wu = _operand(_rows(x, K)), _operand(weight_gate), _operand(weight_up)
    bg, bu = (None if b is None else b.resolve_neg().contiguous() for b in (bias_gate, bias_up))
    M = xk.size(0)
    y = torch.empty(*x.shape[:-1], N, device=dev, dtype=x.dtype)
    factors = torch.empty(_planes(x.dtype), M, N, device=dev, dtype=torch.int16) if save else None
    lib = _lib.load()
    with _device_guard(dev):
        nbytes = lib.fmx_gated_workspace_bytes(M, N, K)
        ws = _lib.workspace(nbytes, dev)
        rc = lib.fmx_gated(
            _lib.dtype_code(xk), xk.data_ptr(), xk.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0),
            _lib.ptr(bg), _lib.ptr(bu), act, M, N, K, y.data_ptr(), _lib.ptr(factors), _lib.ptr(ws), nbytes,
            _lib.stream_of(x),
        )
    _lib.check(rc)
    return y, xk, wg, wu, factors


class _GatedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight_gate, weight_up, bias_gate, bias_up, act):
        need_x, need_g, need_u = ctx.needs_input_grad[:3]
        y, xk, wg, wu, factors = _forward(x, weight_gate, weight_up, bias_gate, bias_up, act, True)
        # dx reads the weights, their gradients read x: an operand that no wanted gradient needs is free to go or to change
        ctx.save_for_backward(xk if need_g or need_u else None, wg if need_x else None, wu if need_x else None, factors)
        ctx.shape, ctx.sizes = x.shape, (xk.size(0), *weight_gate.shape)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _lib.native().refuse_capture(ctx)
        *operands, factors = ctx.saved_tensors
        # hooks on saved tensors may give them back in another layout
        xk, wg, wu = (None if t is None else _operand(t) for t in operands)
        factors = factors.contiguous()
        (M, N, K), dev = ctx.sizes, dy.device
        shapes = ctx.shape, (N, K), (N, K), (N,), (N,)
        grads = [torch.empty(s, device=dev, dtype=dy.dtype) if need else None
                 for s, need in zip(shapes, ctx.needs_input_grad)]
        dys = _rows(dy, N)
        lib = _lib.load()
        with _device_guard(dev):
            nbytes = lib.fmx_gated_bwd_workspace_bytes(M, N, K)
            ws = _lib.workspace(nbytes, dev)
            rc = lib.fmx_gated_bwd(
                _lib.dtype_code(dy), _lib.ptr(xk), 0 if xk is None else xk.stride(0), _lib.ptr(wg),
                0 if wg is None else wg.stride(0), _lib.ptr(wu), 0 if wu is None else wu.stride(0), dys.data_ptr(),
                dys.stride(0), factors.data_ptr(), M, N, K, *map(_lib.ptr, grads), _lib.ptr(ws), nbytes,
                _lib.stream_of(dys),
            )
        _lib.check(rc)
        return *grads, None


def gated_linear(x: torch.Tensor, weight_gate: torch.Tensor, weight_up: torch.Tensor,
                 bias_gate: torch.Tensor | None = None, bias_up: torch.Tensor | None = None,
                 activation: str | None = "silu") -> torch.Tensor:
    """act(x Wg^T + bias_gate) * (x Wu^T + bias_up): [..., N] in x's type.

    x is [..., K], the weights [N, K], the biases [N]; activation is None, "relu",
    "gelu" (by the normal distribution function), "gelu_tanh" (its tanh form) or
    "silu". Differentiable in x, the weights and the biases.
    """
    out = _lib.native().gated_linear(x, weight_gate, weight_up, bias_gate, bias_up, ACTIVATIONS.get(activation, -1))
    if out is not None:
        return out
    _check(x, weight_gate, weight_up, bias_gate, bias_up, activation)
    act = ACTIVATIONS[activation]
    if _differentiated(x, weight_gate, weight_up, bias_gate, bias_up):
        return _GatedLinearFn.apply(x, weight_gate, weight_up, bias_gate, bias_up, act)
    return _forward(x, weight_gate, weight_up, bias_gate, bias_up, act, False)[0]
