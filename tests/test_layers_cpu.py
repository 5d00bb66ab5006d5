"""Refusals of the trained layers' C ABI and Python functions, without a launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd import _lib
from flash_maxsim_amd.flash_maxsim_optim import _Tensor

FAKE = 0x10000  # non-null and aligned, never dereferenced
INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def linear(lib, **kw):
    a = dict(dtype=1, x=FAKE, xs=64, w=FAKE, ws=64, b=None, r=None, rs=0, act=0, M=10, N=32, K=64, y=FAKE, z=None,
             wk=None, wb=0)
    a.update(kw)
    return lib.fmx_linear(*a.values(), None)


def linear_bwd(lib, **kw):
    a = dict(dtype=1, x=FAKE, xs=64, w=FAKE, ws=64, dy=FAKE, dys=32, z=None, act=0, M=10, N=32, K=64, dx=FAKE, dw=FAKE,
             db=FAKE, wk=None, wb=0)
    a.update(kw)
    return lib.fmx_linear_bwd(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=2), INVALID, "dtype"),
    (dict(act=5), INVALID, "activation"),
    (dict(N=0), INVALID, "sizes"),
    (dict(M=-1), INVALID, "sizes"),
    (dict(xs=60), INVALID, "strides"),
    (dict(K=61, xs=61), INVALID, "strides"),
    (dict(ws=56), INVALID, "strides"),
    (dict(xs=1 << 22), UNSUPPORTED, "strides"),
    (dict(K=1 << 24, xs=1 << 25, ws=1 << 25), UNSUPPORTED, "too large"),
    (dict(M=(1 << 31) - 4095), UNSUPPORTED, "too large"),
    (dict(x=None), INVALID, "non-null"),
    (dict(x=FAKE + 8), INVALID, "16-byte"),
    (dict(y=FAKE + 1), INVALID, "aligned"),
    (dict(r=FAKE, rs=-1), INVALID, "residual"),
    (dict(M=128, N=64, K=65536, xs=65536, ws=65536), WORKSPACE, "workspace"),
])
def test_linear_rejects(lib, kw, code, text):
    assert linear(lib, **kw) == code
    assert text in lib.fmx_last_error().decode()


@pytest.mark.parametrize("kw,code,text", [
    (dict(dys=-1), INVALID, "dy stride"),
    (dict(act=2), INVALID, "slope"),
    (dict(dy=None), INVALID, "non-null"),
    (dict(), WORKSPACE, "workspace"),
    (dict(w=FAKE + 2), INVALID, "16-byte"),
])
def test_linear_bwd_rejects(lib, kw, code, text):
    assert linear_bwd(lib, **kw) == code
    assert text in lib.fmx_last_error().decode()


def test_linear_without_work(lib):
    assert linear(lib, M=0) == 0
    assert linear_bwd(lib, dx=None, dw=None, db=None) == 0
    assert lib.fmx_linear_workspace_bytes(0, 8, 8) == 0 and lib.fmx_linear_bwd_workspace_bytes(0, 8, 8) == 0
    assert lib.fmx_linear_workspace_bytes(16384, 4096, 1024) == 0  # enough tiles: k is not split
    # few outputs of many rows: the parts of k are float32 products of their own
    n, k, m = 128, 2048, 24576
    assert lib.fmx_linear_bwd_workspace_bytes(m, n, k) >= 2 * n * k * 4 + m * n * 2


def test_layer_norm_rejects(lib):
    def call(**kw):
        a = dict(dtype=0, x=FAKE, xs=64, wd=0, w=None, b=None, M=4, d=64, eps=1e-5, y=FAKE, mu=None, rs=None)
        a.update(kw)
        return lib.fmx_layer_norm(*a.values(), None)

    for kw, code, text in [(dict(dtype=7), INVALID, "dtype"), (dict(wd=1), INVALID, "weights"),
                           (dict(d=0), INVALID, "sizes"), (dict(d=65537), UNSUPPORTED, "FMX_MAX_D"),
                           (dict(eps=-1.0), INVALID, "eps"), (dict(eps=float("nan")), INVALID, "eps"),
                           (dict(mu=FAKE), INVALID, "together"), (dict(x=None), INVALID, "non-null"),
                           (dict(x=FAKE + 1), INVALID, "aligned"), (dict(xs=-64), INVALID, "sizes")]:
        assert call(**kw) == code and text in lib.fmx_last_error().decode(), kw
    assert call(M=0, x=None) == 0
    rc = lib.fmx_layer_norm_bwd(0, FAKE, 64, FAKE, 64, 0, None, FAKE, FAKE, 4, 64, FAKE, FAKE, FAKE, None, 0, None)
    assert rc == WORKSPACE
    assert lib.fmx_layer_norm_bwd_workspace_bytes(4, 64) == 2 * 64 * 4
    rc = lib.fmx_layer_norm_bwd(0, FAKE, 64, FAKE, 64, 0, None, None, FAKE, 4, 64, FAKE, None, None, None, 0, None)
    assert rc == INVALID


def test_adamw_rejects(lib):
    def call(pd=2, gd=2, cd=1, bits=32, count=1, step=1, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, **kw):
        f = dict(param=FAKE, grad=FAKE, exp_avg=FAKE, exp_avg_sq=FAKE, exp_avg_scale=None, exp_avg_sq_scale=None,
                 copy=None, n=8)
        f.update(kw)
        t = (_Tensor * 1)(_Tensor(*f.values()))
        return lib.fmx_adamw(pd, gd, cd, bits, ctypes.cast(t, ctypes.c_void_p), count, step, lr, b1, b2, eps, wd, None, None)

    for kw, text in [(dict(pd=5), "dtype"), (dict(bits=16), "state_bits"), (dict(step=0), "step"),
                     (dict(count=-1), "count"), (dict(lr=-1.0), "lr"), (dict(b1=1.0), "betas"), (dict(b2=float("nan")), "betas"),
                     (dict(n=-1), "elements"), (dict(grad=None), "null"), (dict(bits=8), "null"),
                     (dict(param=FAKE + 2), "aligned"), (dict(pd=1, copy=FAKE), "copies"), (dict(copy=FAKE, cd=2), "copies"),
                     (dict(pd=0, gd=1), "gradients"), (dict(copy=FAKE, cd=0, gd=1), "gradients")]:
        assert call(**kw) == INVALID and text in lib.fmx_last_error().decode(), kw
    assert call(count=0) == 0
    assert lib.fmx_adamw_decode(0, None, FAKE, 4, FAKE, None) == INVALID
    assert lib.fmx_adamw_decode(0, None, None, 0, None, None) == 0


def test_python_functions_refuse_cpu_tensors_and_bad_types():
    h = torch.zeros(4, 16, dtype=torch.float16)
    w = torch.zeros(8, 16, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        fm.linear(h, w)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        fm.layer_norm(h)
    with pytest.raises(TypeError):
        fm.linear(h.float(), w.float())
    with pytest.raises(AssertionError):
        fm.linear(h, w[:, :8])
    p = torch.zeros(300)
    m, v = fm.adamw_state(p)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        fm.adamw_step([p], [p], [m], [v], 1)
    m, v = fm.adamw_state(p, 8)
    assert m.codes.dtype == torch.int8 and v.codes.dtype == torch.uint8 and m.scales.shape == (2,)
    with pytest.raises(ValueError):
        fm.adamw_state(p, 4)


@pytest.mark.parametrize("kw,code", [
    (dict(x=None, dw=None), WORKSPACE), (dict(w=None, dx=None), WORKSPACE),
    (dict(x=None, xs=0, w=None, ws=0, dx=None, dw=None), WORKSPACE),  # db alone
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(x=None, dx=None), INVALID), (dict(w=None, dw=None), INVALID),
    (dict(x=None, w=None, dy=None, dx=None, dw=None), INVALID),
    (dict(x=None, w=None, act=2, dx=None, dw=None), INVALID),
    (dict(x=None, dw=None, ws=60), INVALID), (dict(w=None, dx=None, xs=60), INVALID),
])
def test_linear_bwd_takes_the_operands_that_it_reads(lib, kw, code):
    assert linear_bwd(lib, **kw) == code


def test_linear_limit_of_k(lib):
    """Rows hold K rounded up to 8 elements, and their strides are below 2^22."""
    top = (1 << 22) - 8
    assert linear(lib, K=top, xs=top, ws=top) == WORKSPACE and linear_bwd(lib, K=top, xs=top, ws=top) == WORKSPACE
    for call in (linear, linear_bwd):
        assert call(lib, K=top + 1, xs=top + 8, ws=top + 8) == UNSUPPORTED and "strides" in lib.fmx_last_error().decode()
