"""Refusals of the encoder block's C ABI and Python functions, without a launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd import _lib
from flash_maxsim_amd.flash_maxsim_muon import _Matrix

FAKE = 0x10000  # non-null and aligned, never dereferenced
INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(lib, rc, code, text):
    assert rc == code and text in lib.fmx_last_error().decode(), (rc, lib.fmx_last_error().decode())


def gated(lib, **kw):
    a = dict(dtype=1, x=FAKE, xs=64, wg=FAKE, gs=64, wu=FAKE, us=64, bg=None, bu=None, act=4, M=10, N=32, K=64, y=FAKE, f=None,
             wk=None, wb=0)
    a.update(kw)
    return lib.fmx_gated(*a.values(), None)


def gated_bwd(lib, **kw):
    a = dict(dtype=1, x=FAKE, xs=64, wg=FAKE, gs=64, wu=FAKE, us=64, dy=FAKE, dys=32, f=FAKE, M=10, N=32, K=64, dx=FAKE,
             dwg=FAKE, dwu=FAKE, dbg=FAKE, dbu=FAKE, wk=None, wb=0)
    a.update(kw)
    return lib.fmx_gated_bwd(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=2), INVALID, "dtype"), (dict(act=5), INVALID, "activation"), (dict(act=-1), INVALID, "activation"),
    (dict(N=0), INVALID, "sizes"), (dict(M=-1), INVALID, "sizes"), (dict(K=0), INVALID, "sizes"),
    (dict(xs=60), INVALID, "strides"), (dict(gs=56), INVALID, "strides"), (dict(us=63), INVALID, "strides"),
    (dict(K=61, xs=61), INVALID, "strides"), (dict(us=1 << 22), UNSUPPORTED, "strides"),
    (dict(N=1 << 20), UNSUPPORTED, "N="), (dict(M=(1 << 31) - 4095), UNSUPPORTED, "too large"),
    (dict(x=None), INVALID, "non-null"), (dict(wg=None), INVALID, "non-null"), (dict(wu=None), INVALID, "non-null"),
    (dict(wu=FAKE + 8), INVALID, "16-byte"), (dict(y=FAKE + 1), INVALID, "aligned"), (dict(f=FAKE + 1), INVALID, "aligned"),
    (dict(bg=FAKE + 1), INVALID, "aligned"), (dict(M=128, N=64, K=65536, xs=65536, gs=65536, us=65536), WORKSPACE, "workspace"),
])
def test_gated_rejects(lib, kw, code, text):
    refused(lib, gated(lib, **kw), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dys=-1), INVALID, "dy stride"), (dict(f=None), INVALID, "non-null"), (dict(dy=None), INVALID, "non-null"),
    (dict(x=None), INVALID, "non-null"), (dict(wg=None), INVALID, "non-null"), (dict(wu=None), INVALID, "non-null"),
    (dict(x=None, dwg=None), INVALID, "non-null"), (dict(dx=FAKE + 1), INVALID, "aligned"), (dict(dbu=FAKE + 1), INVALID, "aligned"),
    (dict(wg=FAKE + 2), INVALID, "16-byte"), (dict(), WORKSPACE, "workspace"), (dict(N=1 << 20), UNSUPPORTED, "N="),
    (dict(x=None, xs=0, dwg=None, dwu=None), WORKSPACE, "workspace"),  # operands that no gradient reads
    (dict(wg=None, gs=0, wu=None, us=0, dx=None), WORKSPACE, "workspace"),
    (dict(x=None, wg=None, wu=None, xs=0, gs=0, us=0, dx=None, dwg=None, dwu=None), WORKSPACE, "workspace"),
])
def test_gated_bwd_rejects(lib, kw, code, text):
    refused(lib, gated_bwd(lib, **kw), code, text)


def test_gated_without_work(lib):
    assert gated(lib, M=0) == 0
    assert gated_bwd(lib, dx=None, dwg=None, dwu=None, dbg=None, dbu=None) == 0
    assert lib.fmx_gated_workspace_bytes(0, 8, 8) == 0 and lib.fmx_gated_bwd_workspace_bytes(0, 8, 8) == 0
    assert lib.fmx_gated_bwd_workspace_bytes(1000, 100, 64) >= 1000 * 2 * 128 * 2  # dg and du, whole stages


def stream(lib, **kw):
    a = dict(dtype=0, x=FAKE, xs=64, r=FAKE, rs=64, g=None, gs=0, wd=0, w=None, b=None, post=0, pw=None, pb=None, scale=None,
             alpha=1.0, rms=0, eps=1e-5, M=4, d=64, h=FAKE, y=FAKE, stats=None)
    a.update(kw)
    return lib.fmx_residual_norm(*a.values(), None)


def stream_bwd(lib, **kw):
    a = dict(dtype=0, x=FAKE, xs=64, r=FAKE, rs=64, g=None, gs=0, wd=0, w=None, post=0, pw=None, pb=None, scale=None, alpha=1.0,
             rms=0, stats=FAKE, dh=FAKE, dhs=64, dy=FAKE, dys=64, M=4, d=64, dx=FAKE, dr=FAKE, dg=None, dw=FAKE, db=FAKE,
             dscale=None, dpw=None, dpb=None, wk=None, wb=0)
    a.update(kw)
    return lib.fmx_residual_norm_bwd(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=7), INVALID, "dtype"), (dict(wd=1), INVALID, "weights"), (dict(d=0), INVALID, "sizes"),
    (dict(M=-1), INVALID, "sizes"), (dict(xs=-1), INVALID, "sizes"), (dict(rs=-1), INVALID, "sizes"),
    (dict(g=FAKE, gs=-1), INVALID, "sizes"), (dict(d=8193), UNSUPPORTED, "MAX_D"), (dict(eps=-1.0), INVALID, "eps"),
    (dict(eps=float("nan")), INVALID, "eps"), (dict(alpha=float("inf")), INVALID, "alpha"), (dict(pw=FAKE), INVALID, "not wanted"),
    (dict(x=None), INVALID, "non-null"), (dict(r=None), INVALID, "non-null"), (dict(h=None), INVALID, "non-null"),
    (dict(y=None), INVALID, "non-null"), (dict(x=FAKE + 1), INVALID, "aligned"), (dict(scale=FAKE + 1), INVALID, "aligned"),
    (dict(wd=2, w=FAKE + 2), INVALID, "aligned"), (dict(stats=FAKE + 8), INVALID, "16-byte"),
])
def test_residual_norm_rejects(lib, kw, code, text):
    refused(lib, stream(lib, **kw), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dhs=-1), INVALID, "strides"), (dict(dys=-1), INVALID, "strides"), (dict(dpw=FAKE), INVALID, "not there"),
    (dict(dg=FAKE), INVALID, "not there"), (dict(stats=None), INVALID, "non-null"), (dict(dh=None, dy=None), INVALID, "non-null"),
    (dict(dy=None), INVALID, "dw and db"), (dict(x=None), INVALID, "non-null"), (dict(dx=FAKE + 1), INVALID, "aligned"),
    (dict(wd=2, dw=FAKE + 2), INVALID, "aligned"), (dict(), WORKSPACE, "workspace"), (dict(d=8193), UNSUPPORTED, "MAX_D"),
    (dict(stats=FAKE + 4), INVALID, "16-byte"),
])
def test_residual_norm_bwd_rejects(lib, kw, code, text):
    refused(lib, stream_bwd(lib, **kw), code, text)


def test_residual_norm_without_work(lib):
    assert stream(lib, M=0, x=None) == 0
    assert stream_bwd(lib, dx=None, dr=None, dw=None, db=None) == 0
    assert lib.fmx_residual_norm_bwd_workspace_bytes(4, 64) == 5 * 64 * 4
    assert lib.fmx_residual_norm_bwd_workspace_bytes(0, 64) == lib.fmx_residual_norm_bwd_workspace_bytes(4, 8193) == 0


def embedding(lib, **kw):
    a = dict(dtype=0, ids=FAKE, bits=64, w=FAKE, ws=64, scale=1.0, T=10, V=100, d=64, y=FAKE)
    a.update(kw)
    return lib.fmx_embedding(*a.values(), None)


def embedding_bwd(lib, **kw):
    a = dict(dtype=0, ids=FAKE, bits=64, dy=FAKE, dys=64, scale=1.0, padding=-1, T=10, V=100, d=64, dw=FAKE, wk=None, wb=0)
    a.update(kw)
    return lib.fmx_embedding_bwd(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=3), INVALID, "dtype"), (dict(bits=16), INVALID, "bits"), (dict(T=-1), INVALID, "sizes"), (dict(V=0), INVALID, "sizes"),
    (dict(d=0), INVALID, "sizes"), (dict(scale=float("nan")), INVALID, "scale"), (dict(T=(1 << 26) + 1), UNSUPPORTED, "large"),
    (dict(V=(1 << 28) + 1), UNSUPPORTED, "large"), (dict(d=65537), UNSUPPORTED, "large"), (dict(ids=None), INVALID, "non-null"),
    (dict(ids=FAKE + 4), INVALID, "aligned"),
])
def test_embedding_rejects(lib, kw, code, text):
    refused(lib, embedding(lib, **kw), code, text)
    refused(lib, embedding_bwd(lib, **kw), code, text)


def test_embedding_pointers_and_work(lib):
    refused(lib, embedding(lib, ws=-1), INVALID, "stride")
    refused(lib, embedding(lib, w=None), INVALID, "non-null")
    refused(lib, embedding(lib, y=FAKE + 1), INVALID, "aligned")
    refused(lib, embedding_bwd(lib, dys=-1), INVALID, "stride")
    refused(lib, embedding_bwd(lib, dw=None), INVALID, "non-null")
    refused(lib, embedding_bwd(lib, dy=FAKE + 1), INVALID, "aligned")
    refused(lib, embedding_bwd(lib), WORKSPACE, "workspace")
    need = lib.fmx_embedding_bwd_workspace_bytes(0, 10, 100, 64)
    refused(lib, embedding_bwd(lib, wk=FAKE + 64, wb=need), WORKSPACE, "256-byte")
    assert embedding(lib, T=0, ids=None, y=None) == 0 and lib.fmx_embedding_bwd_workspace_bytes(0, 0, 100, 64) == 0
    assert lib.fmx_embedding_bwd_workspace_bytes(0, 10, 0, 64) == 0


def muon(lib, step=True, pd=2, gd=2, cd=1, count=1, lr=1e-3, mu=0.95, wd=0.0, steps=5, a=3.4, b=-4.7, c=2.0, eps=1e-7, wk=None,
         wb=0, **kw):
    f = dict(param=FAKE, grad=FAKE, momentum=FAKE, copy=None, rows=8, cols=16)
    f.update(kw)
    t = (_Matrix * 1)(_Matrix(*f.values()))
    if step:
        return lib.fmx_muon(pd, gd, cd, ctypes.cast(t, ctypes.c_void_p), count, lr, mu, 1, wd, steps, a, b, c, eps, 0, None, wk,
                            wb, None)
    return lib.fmx_orthogonalize(pd, gd, ctypes.cast(t, ctypes.c_void_p), count, steps, a, b, c, eps, wk, wb, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(pd=5), INVALID, "dtype"), (dict(count=-1), INVALID, "count"), (dict(lr=-1.0), INVALID, "lr"), (dict(mu=1.0), INVALID, "momentum"),
    (dict(wd=float("nan")), INVALID, "weight_decay"), (dict(steps=0), INVALID, "steps"), (dict(steps=101), INVALID, "steps"),
    (dict(eps=0.0), INVALID, "eps"), (dict(a=float("nan")), INVALID, "coefficients"), (dict(b=-20.5), INVALID, "coefficients"),
    (dict(rows=-1), INVALID, "elements"), (dict(rows=16385, cols=16385), UNSUPPORTED, "sides"),
    (dict(cols=(1 << 20) + 1), UNSUPPORTED, "sides"), (dict(param=None), INVALID, "null"), (dict(grad=None), INVALID, "null"),
    (dict(momentum=None), INVALID, "null"), (dict(param=FAKE + 2), INVALID, "aligned"), (dict(momentum=FAKE + 2), INVALID, "aligned"),
    (dict(pd=1, copy=FAKE), INVALID, "copies"), (dict(copy=FAKE, cd=2), INVALID, "copies"), (dict(pd=0, gd=1), INVALID, "gradients"),
    (dict(copy=FAKE, cd=0, gd=1), INVALID, "gradients"), (dict(), WORKSPACE, "workspace"), (dict(wk=FAKE, wb=8), WORKSPACE, "workspace"),
])
def test_muon_rejects(lib, kw, code, text):
    refused(lib, muon(lib, **kw), code, text)


def test_orthogonalize_rejects(lib):
    for kw, code, text in [(dict(gd=9), INVALID, "dtype"), (dict(steps=0), INVALID, "steps"), (dict(param=None), INVALID, "null"),
                           (dict(c=1e9), INVALID, "coefficients"), (dict(momentum=None), WORKSPACE, "workspace")]:
        refused(lib, muon(lib, False, **kw), code, text)


def test_muon_without_work(lib):
    assert muon(lib, count=0) == 0 and muon(lib, rows=0, param=None) == 0 and muon(lib, False, cols=0, grad=None) == 0
    assert lib.fmx_muon_workspace_bytes(None, 1) == 0
    t = (_Matrix * 2)(_Matrix(None, None, None, None, 100, 300), _Matrix(None, None, None, None, 0, 5))
    # X twice and its lower halves, A and B, of sides rounded up to 64; the sums of squares
    assert lib.fmx_muon_workspace_bytes(t, 2) >= (3 * 128 * 320 + 2 * 128 * 128) * 2 + 8


def test_python_functions_refuse_cpu_tensors_and_bad_arguments():
    h = torch.zeros(4, 16, dtype=torch.float16)
    w = torch.zeros(8, 16, dtype=torch.float16)
    for f in (lambda: fm.gated_linear(h, w, w), lambda: fm.residual_norm(h, h), lambda: fm.embedding(torch.zeros(3, dtype=torch.int64), w),
              lambda: fm.orthogonalize(w), lambda: fm.muon_step([w], [w], [w.float()])):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            f()
    with pytest.raises(TypeError):
        fm.gated_linear(h.float(), w.float(), w.float())
    with pytest.raises(AssertionError):
        fm.gated_linear(h, w, w[:, :8])
    with pytest.raises(ValueError):
        fm.gated_linear(h, w, w, activation="glu")
    with pytest.raises(ValueError):
        fm.residual_norm(h, h, norm="group")
    with pytest.raises(ValueError):
        fm.residual_norm(h, h, post_bias=h[0])
    with pytest.raises(ValueError):
        fm.embedding(torch.zeros(3, dtype=torch.int64), w, padding_idx=8)
    with pytest.raises(ValueError):
        fm.muon_step([w], [w], [])
    with pytest.raises(ValueError):
        fm.Muon([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError):
        fm.Muon([torch.nn.Parameter(torch.zeros(3, 4))], momentum=1.0)
