"""The step between two blocks of an encoder on MI355X, differentiable: add and normalise in one pass.

A block's output x, itself normalised where the block ends in a norm, times a gate
and a learned scale, is added to the hidden states; the next block reads their norm.
Extension of the reference API (no counterpart in flash_maxsim 0.1.0, whose
training starts at the token embeddings).

Rows are float16, bfloat16 or float32; sums, means and deviations are float32, and
h, y and every gradient are rounded once: y is the norm of h before its rounding.
Weights, biases and the scale are of the rows' type or all float32, and so are
their gradients, which are float32 sums in a fixed order: the same inputs give
the same bits.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .flash_maxsim import _check_devices, _device_guard
from .flash_maxsim_norm import _CODES, _differentiated, _rows

NORMS = {"layer": 0, "rms": 1}
MAX_D = 8192


def _weight_type(x, vectors) -> torch.dtype:
    types = {t.dtype for t in vectors if t is not None}
    if not types:
        return x.dtype
    if len(types) > 1 or not types <= {x.dtype, torch.float32}:
        raise TypeError(f"weights, biases and scale must all be {x.dtype} or all float32, got {sorted(map(str, types))}")
    return types.pop()


def _check(x, residual, gate, vectors, norm, post_norm, post_weight, post_bias, residual_scale) -> None:
    if norm not in NORMS:
        raise ValueError(f"norm={norm!r} must be one of {list(NORMS)}")
    if not post_norm and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias need post_norm=True")
    if not math.isfinite(residual_scale):
        raise ValueError(f"residual_scale={residual_scale} must be finite")
    assert x.ndim >= 1 and x.size(-1) >= 1, "x must be [..., d] with d >= 1"
    d = x.size(-1)
    for t in (residual, gate):
        assert t is None or t.shape == x.shape, "residual and gate must have x's shape"
    for t in vectors:
        assert t is None or tuple(t.shape) == (d,), f"weights, biases and scale must be [{d}]"
    if x.dtype not in _CODES:
        raise TypeError(f"x must be float16, bfloat16 or float32, got {x.dtype}")
    for t in (residual, gate):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"residual and gate must be {x.dtype}, got {t.dtype}")


def _vector(t):
    return None if t is None else t.resolve_neg().contiguous()


def _forward(x, residual, gate, weight, bias, post_weight, post_bias, scale, post, alpha, rms, eps, save):
    """h, y, the operands as the kernels read them, and with `save` both norms' float32 mean and inverse deviation."""
    d = x.size(-1)
    dev = _check_devices(x, residual, gate, weight, bias, post_weight, post_bias, scale)
    wt = _weight_type(x, (weight, bias, post_weight, post_bias, scale))
    xr, rr, gr = _rows(x, d), _rows(residual, d), None if gate is None else _rows(gate, d)
    weight, bias, post_weight, post_bias, scale = map(_vector, (weight, bias, post_weight, post_bias, scale))
    M = xr.size(0)
    h, y = (torch.empty(x.shape, device=dev, dtype=x.dtype) for _ in range(2))
    stats = torch.empty(M, 4, device=dev, dtype=torch.float32) if save else None
    with _device_guard(dev):
        rc = _lib.load().fmx_residual_norm(
            _CODES[x.dtype], xr.data_ptr(), xr.stride(0), rr.data_ptr(), rr.stride(0), _lib.ptr(gr),
            0 if gr is None else gr.stride(0), _CODES[wt], _lib.ptr(weight), _lib.ptr(bias), int(post),
            _lib.ptr(post_weight), _lib.ptr(post_bias), _lib.ptr(scale), alpha, rms, eps, M, d, h.data_ptr(),
            y.data_ptr(), _lib.ptr(stats), _lib.stream_of(x),
        )
    _lib.check(rc)
    return h, y, (xr, rr, gr, weight, post_weight, post_bias, scale, stats)


class _ResidualNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gate, weight, bias, post_weight, post_bias, scale, post, alpha, rms, eps):
        h, y, saved = _forward(x, residual, gate, weight, bias, post_weight, post_bias, scale, post, alpha, rms, eps, True)
        ctx.save_for_backward(*saved)
        ctx.set_materialize_grads(False)
        ctx.wt = _weight_type(x, (weight, bias, post_weight, post_bias, scale))
        ctx.shape, ctx.how = x.shape, (post, alpha, rms)
        return h, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dy):
        if dh is None and dy is None:
            return (None,) * 12
        _lib.native().refuse_capture(ctx)
        x, r, g, w, pw, pb, scale, stats = ctx.saved_tensors
        d, (post, alpha, rms) = ctx.shape[-1], ctx.how
        # hooks on saved tensors may give them back in another layout
        x, r, g = (None if t is None else _rows(t, d) for t in (x, r, g))
        w, pw, pb, scale, stats = map(_vector, (w, pw, pb, scale, stats))
        M, dev = x.size(0), x.device
        dhs, dys = (None if t is None else _rows(t, d) for t in (dh, dy))
        need = list(ctx.needs_input_grad[:8])
        if dy is None:  # w and b have no part in h
            need[3] = need[4] = False
        rows = [torch.empty(ctx.shape, device=dev, dtype=x.dtype) if n else None for n in need[:3]]
        dw, db, dpw, dpb, dscale = (torch.empty(d, device=dev, dtype=ctx.wt) if n else None for n in need[3:])
        lib = _lib.load()
        with _device_guard(dev):
            nbytes = lib.fmx_residual_norm_bwd_workspace_bytes(M, d) if any(need[3:]) else 0
            ws = _lib.workspace(nbytes, dev)
            rc = lib.fmx_residual_norm_bwd(
                _CODES[x.dtype], x.data_ptr(), x.stride(0), r.data_ptr(), r.stride(0), _lib.ptr(g),
                0 if g is None else g.stride(0), _CODES[ctx.wt], _lib.ptr(w), int(post), _lib.ptr(pw), _lib.ptr(pb),
                _lib.ptr(scale), alpha, rms, stats.data_ptr(), _lib.ptr(dhs), 0 if dhs is None else dhs.stride(0),
                _lib.ptr(dys), 0 if dys is None else dys.stride(0), M, d, *map(_lib.ptr, rows), _lib.ptr(dw),
                _lib.ptr(db), _lib.ptr(dscale), _lib.ptr(dpw), _lib.ptr(dpb), _lib.ptr(ws), nbytes, _lib.stream_of(x),
            )
        _lib.check(rc)
        return *rows, dw, db, dpw, dpb, dscale, None, None, None, None


def residual_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, *, norm: str = "layer", eps: float = 1e-5, post_norm: bool = False,
                  post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                  residual_scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(h, y): h = residual_scale * residual + scale * gate * post(x) and y = norm(h) * weight + bias.

    x, residual and gate are [..., d] with d from 1 to 8192; weight, bias,
    post_weight, post_bias and scale are [d]. post(x) is x, or with post_norm
    norm(x) * post_weight + post_bias. norm is "layer" (mean removed, the biased
    variance) or "rms"; both norms are of one kind. What is None is one (a bias: zero). h and y
    have x's shape and type; differentiable in all tensors.
    """
    vectors = weight, bias, post_weight, post_bias, scale
    if norm in NORMS and math.isfinite(residual_scale):
        out = _lib.native().residual_norm(x, residual, gate, *vectors, post_norm, float(residual_scale), NORMS[norm], eps)
        if out is not None:
            return out
    _check(x, residual, gate, vectors, norm, post_norm, post_weight, post_bias, residual_scale)
    args = (x, residual, gate, *vectors, bool(post_norm), float(residual_scale), NORMS[norm], float(eps))
    if _differentiated(x, residual, gate, *vectors):
        return _ResidualNormFn.apply(*args)
    h, y, _ = _forward(*args, False)
    return h, y
