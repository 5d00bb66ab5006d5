"""AdamW on MI355X: one pass over all tensors, moments in float32 or 8 bits.

What moves the weights of the layers trained through flash_maxsim_train.
Extension of the reference API (no counterpart in flash_maxsim 0.1.0).

adamw_step updates lists of tensors in place; AdamW is the optimizer class over
it. Parameters are float32, float16 or bfloat16, gradients of the same type or
float32; arithmetic is float32 and each parameter is rounded once. float32
parameters can have 16-bit copies, written in the same pass, for the next
forward.

8-bit moments (AdamW8bitState) hold one byte a value and one float32 scale for
every 256 consecutive elements of a tensor: the first moment is c |c| scale with
int8 codes c, of the second moment the root is held, c^2 scale with uint8 codes.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .flash_maxsim import _check_devices, _device_guard

BLOCK = 256

_CODES = {torch.float16: _lib.FMX_DTYPE_F16, torch.bfloat16: _lib.FMX_DTYPE_BF16, torch.float32: _lib.FMX_DTYPE_F32}


class AdamW8bitState(NamedTuple):
    """A moment in 8 bits: codes (int8 of the first moment, uint8 of the second),
    one per parameter element, and scales, float32, one per 256 of them."""

    codes: torch.Tensor
    scales: torch.Tensor


class _Tensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale",
                                               "exp_avg_sq_scale", "copy")] + [("n", ctypes.c_int64)]


def adamw_state(param: torch.Tensor, bits: int = 32):
    """(exp_avg, exp_avg_sq) of zeros for a parameter: float32 tensors, or
    AdamW8bitState pairs when bits is 8."""
    if bits == 32:
        return (torch.zeros(param.shape, dtype=torch.float32, device=param.device),
                torch.zeros(param.shape, dtype=torch.float32, device=param.device))
    if bits != 8:
        raise ValueError(f"bits={bits} must be 8 or 32")
    blocks = -(-param.numel() // BLOCK)
    return tuple(AdamW8bitState(torch.zeros(param.shape, dtype=t, device=param.device),
                                torch.zeros(blocks, dtype=torch.float32, device=param.device))
                 for t in (torch.int8, torch.uint8))


def dequantize_adamw(state: AdamW8bitState) -> torch.Tensor:
    """The float32 values of an 8-bit moment, in its codes' shape: the first
    moment of int8 codes, the second (the root's square) of uint8 codes."""
    codes, scales = state
    out = _lib.native().adamw_decode(codes, scales)
    if out is not None:
        return out
    if codes.dtype not in (torch.int8, torch.uint8) or scales.dtype != torch.float32:
        raise TypeError(f"an 8-bit moment holds int8 or uint8 codes and float32 scales, got {codes.dtype}, {scales.dtype}")
    assert scales.numel() == -(-codes.numel() // BLOCK), "one scale per 256 codes"
    dev = _check_devices(codes, scales)
    codes, scales = codes.contiguous(), scales.contiguous()
    out = torch.empty(codes.shape, dtype=torch.float32, device=dev)
    with _device_guard(dev):
        rc = _lib.load().fmx_adamw_decode(int(codes.dtype == torch.uint8), codes.data_ptr(), scales.data_ptr(),
                                          codes.numel(), out.data_ptr(), _lib.stream_of(codes))
    _lib.check(rc)
    return out


def _moment(s, p, eight: bool, codes: torch.dtype):
    """(values or codes, scales or None) of one moment, checked against its parameter."""
    if isinstance(s, tuple) != eight:
        raise ValueError("every moment of a step is held in the same number of bits")
    data, scales = (s[0], s[1]) if eight else (s, None)
    want = codes if eight else torch.float32
    if data.dtype != want:
        raise TypeError(f"expected a moment in {want}, got {data.dtype}")
    if data.numel() != p.numel() or not data.is_contiguous():
        raise ValueError("a moment has its parameter's number of elements and is contiguous")
    if eight:
        if scales.dtype != torch.float32:
            raise TypeError(f"scales must be float32, got {scales.dtype}")
        if scales.numel() != -(-p.numel() // BLOCK) or not scales.is_contiguous():
            raise ValueError(f"scales must be contiguous, one for each {BLOCK} elements")
    return data, scales


def _step_python(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps, weight_decay, grad_scale, copies) -> None:
    lists = [list(x) for x in (params, grads, exp_avgs, exp_avg_sqs)]
    params, grads, exp_avgs, exp_avg_sqs = lists
    copies = [None] * len(params) if copies is None else list(copies)
    if any(len(x) != len(params) for x in (*lists, copies)):
        raise ValueError("params, grads, exp_avgs, exp_avg_sqs and copies must have the same length")
    if grad_scale is not None:
        assert grad_scale.numel() == 1, "grad_scale is one value"
        if grad_scale.dtype != torch.float32:
            raise TypeError(f"grad_scale must be float32, got {grad_scale.dtype}")
    if not params:
        return
    eight = isinstance(exp_avgs[0], tuple)
    batches: dict = {}
    keep = []  # contiguous copies of gradients, until the launches
    for p, g, m, v, c in zip(params, grads, exp_avgs, exp_avg_sqs, copies):
        if p.dtype not in _CODES:
            raise TypeError(f"parameters must be float16, bfloat16 or float32, got {p.dtype}")
        if c is not None and (p.dtype != torch.float32 or c.dtype not in (torch.float16, torch.bfloat16)):
            raise TypeError(f"copies are float16 or bfloat16, of float32 parameters; got {c.dtype} of {p.dtype}")
        # a 16-bit gradient of a float32 parameter is of its copy's type, where it has one
        if g.dtype not in (p.dtype, torch.float32) and not (p.dtype == torch.float32 and g.dtype in _CODES and
                                                            (c is None or c.dtype == g.dtype)):
            raise TypeError(f"gradients must be float32 or of their parameters' (or copies') type, got {g.dtype} for {p.dtype}")
        assert g.shape == p.shape and (c is None or c.shape == p.shape), "a gradient (copy) has its parameter's shape"
        if any(t is not None and (t.is_neg() or not t.is_contiguous()) for t in (p, c)):
            raise ValueError("parameters and copies must be contiguous: they are written in place")
        m, ms = _moment(m, p, eight, torch.int8)
        v, vs = _moment(v, p, eight, torch.uint8)
        dev = _check_devices(p, g, m, v, ms, vs, c, grad_scale)
        if g.is_neg() or not g.is_contiguous():
            g = g.resolve_neg().contiguous()
            keep.append(g)
        row = _Tensor(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), _lib.ptr(ms), _lib.ptr(vs), _lib.ptr(c),
                      p.numel())
        batches.setdefault((dev, p.dtype, g.dtype, None if c is None else c.dtype), []).append(row)
    lib = _lib.load()
    for (dev, pt, gt, ct), rows in batches.items():
        table = (_Tensor * len(rows))(*rows)
        with _device_guard(dev):
            rc = lib.fmx_adamw(_CODES[pt], _CODES[gt], _CODES[ct or torch.bfloat16], 8 if eight else 32, table,
                               len(rows), step, lr, *betas, eps, weight_decay, _lib.ptr(grad_scale),
                               torch.cuda.current_stream(dev).cuda_stream)
        _lib.check(rc)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step: int, lr: float = 1e-3, betas=(0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 0.01, grad_scale: torch.Tensor | None = None,
               copies=None) -> None:
    """One AdamW step (decoupled weight decay) over lists of tensors, in place.

    exp_avgs and exp_avg_sqs hold the moments of each parameter: float32 tensors,
    or AdamW8bitState pairs (codes, scales), all of one kind (adamw_state makes
    either). `step`
    counts from 1. grad_scale, a float32 value on the GPU, multiplies every
    gradient (a clipping factor, the inverse of a loss scale) without a read back.
    copies, a list with a float16 or bfloat16 tensor (or None) for each
    parameter, receives the new float32 parameters rounded.
    """
    step, betas = int(step), (float(betas[0]), float(betas[1]))
    lr, eps, weight_decay = float(lr), float(eps), float(weight_decay)
    if _lib.native().adamw(params, grads, exp_avgs, exp_avg_sqs, step, lr, *betas, eps, weight_decay, grad_scale, copies):
        return
    params = list(params)
    copies = None if copies is None else list(copies)
    _step_python(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps, weight_decay, grad_scale, copies)
    torch.autograd.graph.increment_version(params if copies is None else params + [c for c in copies if c is not None])


class AdamW(torch.optim.Optimizer):
    """AdamW over adamw_step: all of a group's tensors in one pass.

    state_bits is 32 or 8. copies, in the order of the parameters, are 16-bit
    tensors (or None) that receive the new float32 parameters. Learning-rate
    schedulers, parameter groups and state_dict work as with torch's optimizers;
    loaded moments stay in the bits they have. `step(grad_scale=...)` passes a float32 GPU
    scalar that multiplies the gradients.
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                 state_bits: int = 32, copies=None):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits={state_bits} must be 8 or 32")
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and all(0 <= b < 1 for b in betas)):
            raise ValueError("lr, eps and weight_decay must be >= 0, betas in [0, 1)")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self._bits = state_bits
        mine = [p for g in self.param_groups for p in g["params"]]
        copies = [None] * len(mine) if copies is None else list(copies)
        if len(copies) != len(mine):
            raise ValueError(f"{len(copies)} copies for {len(mine)} parameters")
        self._copies = {id(p): c for p, c in zip(mine, copies) if c is not None}

    def __getstate__(self):
        """torch's, with the bits and the copies (deep copies and pickles)."""
        params = [p for g in self.param_groups for p in g["params"]]
        return super().__getstate__() | {"_bits": self._bits, "_copies": [self._copies.get(id(p)) for p in params]}

    def __setstate__(self, state) -> None:
        """torch calls this too when it loads a state_dict, whose state has neither."""
        copies = state.get("_copies")
        super().__setstate__({k: v for k, v in state.items() if k != "_copies"})
        if copies is not None:
            params = [p for g in self.param_groups for p in g["params"]]
            self._copies = {id(p): c for p, c in zip(params, copies) if c is not None}

    @torch.no_grad()
    def step(self, closure=None, grad_scale: torch.Tensor | None = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            batches: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                s = self.state[p]
                if not s:
                    m, v = adamw_state(p, self._bits)
                    s["step"] = 0
                    if self._bits == 8:
                        s["exp_avg"], s["exp_avg_scale"] = m
                        s["exp_avg_sq"], s["exp_avg_sq_scale"] = v
                    else:
                        s["exp_avg"], s["exp_avg_sq"] = m, v
                s["step"] += 1
                eight = "exp_avg_scale" in s  # loaded 32-bit moments may stand beside new 8-bit ones
                row = batches.setdefault((s["step"], eight), ([], [], [], [], []))
                row[0].append(p)
                row[1].append(p.grad)
                if eight:
                    row[2].append(AdamW8bitState(s["exp_avg"], s["exp_avg_scale"]))
                    row[3].append(AdamW8bitState(s["exp_avg_sq"], s["exp_avg_sq_scale"]))
                else:
                    row[2].append(s["exp_avg"])
                    row[3].append(s["exp_avg_sq"])
                row[4].append(self._copies.get(id(p)))
            for (step, _), (p, g, m, v, c) in batches.items():
                adamw_step(p, g, m, v, step, group["lr"], group["betas"], group["eps"], group["weight_decay"],
                           grad_scale, c if any(x is not None for x in c) else None)
        return loss

    def load_state_dict(self, state_dict) -> None:
        """torch's, with moments and scales in float32 and codes in their type again (torch casts
        float state to its parameter's type, which would round the moments). A state of
        torch.optim.AdamW, whose moments of 16-bit parameters are 16-bit, continues as one of 32 bits."""
        if any(g.get("amsgrad") or g.get("maximize") for g in state_dict["param_groups"]):
            raise ValueError("this AdamW has neither amsgrad nor maximize")
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        super().load_state_dict(state_dict)
        mine = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, mine):
            for k, v in saved.get(i, {}).items():
                if k == "step":  # a tensor in states of torch's optimizers
                    self.state[p][k] = int(v)
                elif torch.is_tensor(v):  # codes keep their type; torch's moments are of the parameters'
                    dtype = torch.float32 if v.is_floating_point() else v.dtype
                    self.state[p][k] = v.detach().to(p.device, dtype, copy=True).contiguous()
                else:
                    self.state[p][k] = v
