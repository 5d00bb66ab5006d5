"""Orthogonalised updates of weight matrices on MI355X, as the Muon optimiser makes them.

What moves the matrices of the layers trained through flash_maxsim_train, beside
AdamW for vectors and tables. Extension of the reference API (no counterpart in
flash_maxsim 0.1.0).

The momentum's matrix is divided by its norm, and every singular value s of it
goes to a s + b s^3 + c s^5 a few times, which brings all of them near one: three
products a step on matrix instructions, over all matrices in one launch. Products
take fp16 operands and float32 sums; the iterate is held as a pair of fp16
values, so that small singular values, which grow by hundreds, do not drown in
its rounding. The result is within about 2.5e-3 (of its norm) of the formula's where the
shorter side is 16 or more; of shorter ones, whose few singular values' errors do not
average out, the median is 2e-3 and the worst of some thousands 1.4e-2.
Sums have a fixed order: the same inputs give the same bits.

muon_step updates lists of matrices in place; Muon is the optimizer class over
it. Parameters are float32, float16 or bfloat16, gradients of the same type or
float32, momenta float32; each parameter is rounded once. float32 parameters can
have 16-bit copies, written in the same pass, for the next forward.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .flash_maxsim import _check_devices, _device_guard

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_SHORT, MAX_LONG = 1 << 14, 1 << 20
ADJUST = {"original": 0, "match_rms_adamw": 1}

_CODES = {torch.float16: _lib.FMX_DTYPE_F16, torch.bfloat16: _lib.FMX_DTYPE_BF16, torch.float32: _lib.FMX_DTYPE_F32}


class _Matrix(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "momentum", "copy")] + [("rows", ctypes.c_int64),
                                                                                      ("cols", ctypes.c_int64)]


def _coefficients(c) -> tuple[float, float, float]:
    c = tuple(float(x) for x in c)
    if len(c) != 3:
        raise ValueError(f"coefficients are three numbers, got {len(c)}")
    return c


def _workspace(lib, table, count: int, dev) -> tuple[torch.Tensor | None, int]:
    nbytes = lib.fmx_muon_workspace_bytes(table, count)
    return _lib.workspace(nbytes, dev), nbytes


def _check_sides(t: torch.Tensor) -> None:
    if min(t.shape) > MAX_SHORT or max(t.shape) > MAX_LONG:
        raise ValueError(f"a matrix of {tuple(t.shape)}: its sides are at most {MAX_SHORT} and {MAX_LONG}")


def _apart(written, read) -> None:
    """No memory that is written is also another tensor's: a step reads gradients and their scale again after it has
    written momenta."""
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), w)
             for ts, w in ((written, True), (read, False)) for t in ts if t.numel() and t.is_contiguous()]
    end, end_written = 0, 0  # of all before, and of those that are written
    for first, last, w in sorted(spans):
        if first < (end if w else end_written):
            raise ValueError("params, momenta and copies must not share memory with each other, with gradients or grad_scale")
        end, end_written = max(end, last), max(end_written, last) if w else end_written


def _no_tangents(tensors) -> None:
    if torch.autograd.forward_ad._current_level >= 0 and any(
            torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("flash_maxsim_amd: no forward-mode derivative of an optimizer's step")


@torch.no_grad()
def orthogonalize(updates, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7):
    """The orthogonalised matrices of updates (a 2-D tensor, or a list of them), in their types and shapes.

    Each is divided by the root of its squares' sum (at least eps), then
    X = a X + (b X X^T + c (X X^T)^2) X `steps` times with (a, b, c) =
    coefficients, each within +-20. Types may differ from matrix to matrix. No gradients.
    """
    one = isinstance(updates, torch.Tensor)
    updates = [updates] if one else list(updates)
    _no_tangents(updates)
    steps, coefficients, eps = int(steps), _coefficients(coefficients), float(eps)
    out: list = [None] * len(updates)
    batches: dict = {}
    keep = []  # contiguous copies, until the launches
    for i, u in enumerate(updates):
        assert u.ndim == 2, "an update is a matrix"
        _check_sides(u)
        if u.dtype not in _CODES:
            raise TypeError(f"updates must be float16, bfloat16 or float32, got {u.dtype}")
        dev = _check_devices(u)
        if u.is_neg() or not u.is_contiguous():
            u = u.resolve_neg().contiguous()
            keep.append(u)
        out[i] = torch.empty(u.shape, dtype=u.dtype, device=dev)
        row = _Matrix(out[i].data_ptr(), u.data_ptr(), None, None, *u.shape)
        batches.setdefault((dev, u.dtype), []).append(row)
    lib = _lib.load()
    for (dev, dtype), rows in batches.items():
        table = (_Matrix * len(rows))(*rows)
        with _device_guard(dev):
            ws, nbytes = _workspace(lib, table, len(rows), dev)
            rc = lib.fmx_orthogonalize(_CODES[dtype], _CODES[dtype], table, len(rows), steps, *coefficients, eps,
                                       _lib.ptr(ws), nbytes, torch.cuda.current_stream(dev).cuda_stream)
        _lib.check(rc)
    return out[0] if one else out


@torch.no_grad()
def muon_step(params, grads, momenta, lr: float = 1e-3, momentum: float = 0.95, nesterov: bool = True,
              weight_decay: float = 0.1, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7,
              adjust: str = "original", grad_scale: torch.Tensor | None = None, copies=None) -> None:
    """One orthogonalised step over lists of matrices, in place.

    m = momentum m + (1 - momentum) g; what is orthogonalised is m, with nesterov
    (1 - momentum) g + momentum m; then p = p (1 - lr weight_decay) - lr f X with
    f = sqrt(max(1, rows / cols)) (adjust="original") or 0.2 sqrt(max(rows, cols))
    ("match_rms_adamw": steps as large as AdamW's). momenta are float32, of their
    parameters' shapes. grad_scale, a float32 value on the GPU, multiplies every
    gradient without a read back. copies, a list with a float16 or bfloat16 tensor
    (or None) for each parameter, receives the new float32 parameters rounded.
    params, momenta and copies share no memory with each other, with gradients or with grad_scale.
    """
    if adjust not in ADJUST:
        raise ValueError(f"adjust={adjust!r} must be one of {list(ADJUST)}")
    params, grads, momenta = list(params), list(grads), list(momenta)
    copies = [None] * len(params) if copies is None else list(copies)
    if any(len(x) != len(params) for x in (grads, momenta, copies)):
        raise ValueError("params, grads, momenta and copies must have the same length")
    steps, coefficients, eps, lr = int(steps), _coefficients(coefficients), float(eps), float(lr)
    momentum, weight_decay = float(momentum), float(weight_decay)
    if grad_scale is not None:
        assert grad_scale.numel() == 1, "grad_scale is one value"
        if grad_scale.dtype != torch.float32:
            raise TypeError(f"grad_scale must be float32, got {grad_scale.dtype}")
    _no_tangents([*params, *grads, *momenta])
    batches: dict = {}
    keep = []  # contiguous copies of gradients, until the launches
    for p, g, m, c in zip(params, grads, momenta, copies):
        if p.dtype not in _CODES:
            raise TypeError(f"parameters must be float16, bfloat16 or float32, got {p.dtype}")
        if c is not None and (p.dtype != torch.float32 or c.dtype not in (torch.float16, torch.bfloat16)):
            raise TypeError(f"copies are float16 or bfloat16, of float32 parameters; got {c.dtype} of {p.dtype}")
        # a 16-bit gradient of a float32 parameter is of its copy's type, where it has one
        if g.dtype not in (p.dtype, torch.float32) and not (p.dtype == torch.float32 and g.dtype in _CODES and
                                                            (c is None or c.dtype == g.dtype)):
            raise TypeError(f"gradients must be float32 or of their parameters' (or copies') type, got {g.dtype} for {p.dtype}")
        if m.dtype != torch.float32:
            raise TypeError(f"momenta must be float32, got {m.dtype}")
        assert p.ndim == 2, "a parameter is a matrix"
        _check_sides(p)
        assert g.shape == p.shape and m.shape == p.shape and (c is None or c.shape == p.shape), \
            "gradient, momentum and copy have their parameter's shape"
        if any(t is not None and (t.is_neg() or not t.is_contiguous()) for t in (p, m, c)):
            raise ValueError("parameters, momenta and copies must be contiguous: they are written in place")
        dev = _check_devices(p, g, m, c, grad_scale)
        if g.is_neg() or not g.is_contiguous():
            g = g.resolve_neg().contiguous()
            keep.append(g)
        row = _Matrix(p.data_ptr(), g.data_ptr(), m.data_ptr(), _lib.ptr(c), *p.shape)
        batches.setdefault((dev, p.dtype, g.dtype, None if c is None else c.dtype), []).append(row)
    _apart([t for t in (*params, *momenta, *copies) if t is not None], [*grads, *([] if grad_scale is None else [grad_scale])])
    lib = _lib.load()
    for (dev, pt, gt, ct), rows in batches.items():
        table = (_Matrix * len(rows))(*rows)
        with _device_guard(dev):
            ws, nbytes = _workspace(lib, table, len(rows), dev)
            rc = lib.fmx_muon(_CODES[pt], _CODES[gt], _CODES[ct or torch.bfloat16], table, len(rows), lr, momentum,
                              int(nesterov), weight_decay, steps, *coefficients, eps, ADJUST[adjust],
                              _lib.ptr(grad_scale), _lib.ptr(ws), nbytes, torch.cuda.current_stream(dev).cuda_stream)
        _lib.check(rc)
    torch.autograd.graph.increment_version([t for t in (*params, *momenta, *copies) if t is not None])


class Muon(torch.optim.Optimizer):
    """Orthogonalised updates over muon_step: all of a group's matrices in one pass.

    For weight matrices; vectors and embedding tables go to AdamW. copies, in the
    order of the parameters, are 16-bit tensors (or None) that receive the new
    float32 parameters. Learning-rate schedulers, parameter groups and state_dict
    work as with torch's optimizers; the momentum (state "momentum_buffer") is
    float32. `step(grad_scale=...)` passes a float32 GPU scalar that multiplies
    the gradients.
    """

    def __init__(self, params, lr: float = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95, nesterov: bool = True,
                 coefficients=COEFFICIENTS, eps: float = 1e-7, steps: int = 5, adjust: str = "original", copies=None):
        if not (lr >= 0 and weight_decay >= 0 and 0 <= momentum < 1 and eps > 0):
            raise ValueError("lr and weight_decay must be >= 0, momentum in [0, 1), eps > 0")
        if adjust not in ADJUST:
            raise ValueError(f"adjust={adjust!r} must be one of {list(ADJUST)}")
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                                      coefficients=_coefficients(coefficients), eps=eps, steps=steps, adjust=adjust))
        mine = [p for g in self.param_groups for p in g["params"]]
        for p in mine:
            if p.ndim != 2:
                raise ValueError(f"Muon moves matrices, got a parameter of shape {tuple(p.shape)}")
        copies = [None] * len(mine) if copies is None else list(copies)
        if len(copies) != len(mine):
            raise ValueError(f"{len(copies)} copies for {len(mine)} parameters")
        self._copies = {id(p): c for p, c in zip(mine, copies) if c is not None}

    def __getstate__(self):
        """torch's, with the copies (deep copies and pickles)."""
        params = [p for g in self.param_groups for p in g["params"]]
        return super().__getstate__() | {"_copies": [self._copies.get(id(p)) for p in params]}

    def __setstate__(self, state) -> None:
        """torch calls this too when it loads a state_dict, whose state has no copies."""
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
            params = [p for p in group["params"] if p.grad is not None]
            for p in params:
                if "momentum_buffer" not in self.state[p]:
                    self.state[p]["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            copies = [self._copies.get(id(p)) for p in params]
            muon_step(params, [p.grad for p in params], [self.state[p]["momentum_buffer"] for p in params], group["lr"],
                      group["momentum"], group["nesterov"], group["weight_decay"], group["steps"], group["coefficients"],
                      group["eps"], group["adjust"], grad_scale, copies)
        return loss

    def load_state_dict(self, state_dict) -> None:
        """torch's, with the momenta in float32 again (torch casts state to its parameter's type, which would round
        them). A state of torch.optim.Muon continues."""
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        # torch's optimizer of this name has its settings under names of its own
        names = {"ns_coefficients": "coefficients", "ns_steps": "steps", "adjust_lr_fn": "adjust"}
        groups = []
        for g in state_dict["param_groups"]:
            g = {names.get(k, k): v for k, v in g.items()}
            groups.append(g | {"adjust": g.get("adjust") or "original"})
        super().load_state_dict({**state_dict, "param_groups": groups})
        mine = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, mine):
            m = saved.get(i, {}).get("momentum_buffer")
            if torch.is_tensor(m):
                self.state[p]["momentum_buffer"] = m.detach().to(p.device, torch.float32, copy=True).contiguous()
