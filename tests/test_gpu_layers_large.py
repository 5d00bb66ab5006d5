"""The trained layers past 2^32 elements, where 32-bit offsets would wrap, and past a launch's rows."""

from __future__ import annotations

import pytest
import torch

import flash_maxsim_amd as fm

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
U16 = 2.0 ** -11
DEV = "cuda"


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of free GPU memory")
    yield
    torch.cuda.empty_cache()


def filled(M, d, seed):
    """float16 rows whose values repeat every 4099 rows, so that a part tells what every row holds."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    part = torch.randn(4099, d, generator=g, device=DEV).half()
    x = torch.empty(M, d, dtype=torch.float16, device=DEV)
    for a in range(0, M, 4099 * 512):
        n = min(4099 * 512, M - a)
        x[a:a + n] = part.repeat(-(-n // 4099), 1)[:n]
    return x, part


def test_linear():
    M, N, K = (1 << 24) + 777, 8, 264  # x holds 4.4e9 elements; more than 2^24 rows go in two launches
    x, part = filled(M, K, 1)
    g = torch.Generator(device=DEV).manual_seed(2)
    w = (torch.randn(N, K, generator=g, device=DEV) / 16).half().requires_grad_(True)
    b = torch.randn(N, generator=g, device=DEV).half().requires_grad_(True)
    x.requires_grad_(True)
    y = fm.linear(x, w, b, "silu")
    pick = torch.tensor([0, 1, 4098, 4099, 1 << 20, (1 << 24) - 1, 1 << 24, M - 2, M - 1], device=DEV)
    rows = part[pick % 4099].double()
    z = rows @ w.detach().double().t() + b.detach().double()
    want = z * torch.sigmoid(z)
    tol = U16 * want.abs() + 1.13 * F32 * (K + 4) * (rows.abs() @ w.detach().double().abs().t() + 1) + 2.0 ** -20 * z.abs()
    assert ((y.detach()[pick].double() - want).abs() <= tol + 2.0 ** -25).all()
    dy = torch.zeros(M, N, dtype=torch.float16, device=DEV)
    dy[pick] = torch.randn(len(pick), N, generator=g, device=DEV).half()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    s = torch.sigmoid(z)
    dz = dy[pick].double() * s * (1 + z * (1 - s))
    # z and dz rounded to 11 bits, the slope's own slope below 1.13 for arguments of a few units
    near = 4 * U16 * dy[pick].double().abs() * (1 + z.abs())
    assert ((dx[pick].double() - dz @ w.detach().double()).abs() <= near @ w.detach().double().abs() + 2.0 ** -20).all()
    assert not dx[5000].any() and not dx[M - 3].any()
    assert ((dw.double() - dz.t() @ rows).abs() <= near.t() @ rows.abs() + 2 * U16 * (dz.t() @ rows).abs() + 2.0 ** -20).all()
    assert ((db.double() - dz.sum(0)).abs() <= near.sum(0) + U16 * dz.sum(0).abs() + 2.0 ** -20).all()


def test_layer_norm():
    M, d = (1 << 23) + 5, 520
    x, part = filled(M, d, 3)
    x.requires_grad_(True)
    w = torch.linspace(0.5, 1.5, d, device=DEV).half().requires_grad_(True)
    y = fm.layer_norm(x, w)
    pick = torch.tensor([0, 4098, 4099, 1 << 22, M - 2, M - 1], device=DEV)
    rows = part[pick % 4099].double()
    e = rows - rows.mean(1, keepdim=True)
    rs = 1 / torch.sqrt((e * e).mean(1, keepdim=True) + 1e-5)
    xh, wd = e * rs, w.detach().double()
    assert ((y.detach()[pick].double() - xh * wd).abs() <= U16 * (xh * wd).abs() + 1e-5).all()
    dy = torch.zeros(M, d, dtype=torch.float16, device=DEV)
    dy[pick] = torch.randn(len(pick), d, device=DEV).half()
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    g = dy[pick].double() * wd
    want = rs * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    assert ((dx[pick].double() - want).abs() <= U16 * want.abs() + 2e-5).all() and not dx[M - 3].any()
    want = (dy[pick].double() * xh).sum(0)
    assert ((dw.double() - want).abs() <= U16 * want.abs() + 2e-5).all()


def test_adamw():
    n = (1 << 32) + 1027
    p = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([0, 1 << 20, (1 << 31) + 3, (1 << 32) - 1, 1 << 32, n - 1], device=DEV)
    p[at], g[at] = 1.0, 0.5
    m, v = fm.adamw_state(p, 8)
    fm.adamw_step([p], [g], [m], [v], 1, lr=0.25, weight_decay=0.0)
    # the first step is lr times the gradient's sign, exact in bfloat16 but for eps / |g|
    assert ((p[at].double() - 0.75).abs() <= 0.75 * 2.0 ** -8).all()
    assert int((p != 0).sum()) == len(at) and int((m.codes != 0).sum()) == len(at)
    assert (m.codes[at] == 127).all() and (v.codes[at] == 255).all()
    md = fm.dequantize_adamw(m)
    assert ((md[at].double() - 0.05).abs() <= 0.05 * 8 * F32).all()
    del md
    vd = fm.dequantize_adamw(v)
    assert ((vd[at].double() - 0.00025).abs() <= 0.00025 * 2.0 ** -20).all() and int((vd != 0).sum()) == len(at)


@pytest.mark.parametrize("M,N,K", [(512, 4_300_004, 512), (128, 9_000_004, 512), (256, (1 << 24) - 1, 512)])
@pytest.mark.parametrize("name", [None, "relu"])
def test_linear_of_many_outputs(M, N, K, name):
    """dz's rows are N wide: the last row of a tile of 256 (128) lies past 2^31 bytes of its first from N = 4.2 (8.4)
    million on. Few columns of dy are not zero, so dx is a small product."""
    g = torch.Generator(device=DEV).manual_seed(N)
    w = torch.randn(1031, K, generator=g, device=DEV).bfloat16().repeat(-(-N // 1031), 1)[:N].requires_grad_(True)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16().requires_grad_(True)
    pick = torch.tensor([0, 7, 8, 63, 64, N // 3, N // 2, (1 << 22) - 1, 1 << 22, N - 9, N - 1], device=DEV)
    y = fm.linear(x, w, None, name)
    z = x.detach().double() @ w.detach()[pick].double().t()
    dy = torch.zeros(M, N, dtype=torch.bfloat16, device=DEV)
    dy[:, pick] = torch.randn(M, len(pick), generator=g, device=DEV).bfloat16()
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    far = z.abs() > F32 * (K + 4) * (x.detach().double().abs() @ w.detach()[pick].double().abs().t())  # relu's slope jumps at zero
    dz = dy[:, pick].double() * (1.0 if name is None else (z > 0).double())
    loose = torch.zeros_like(dz) if name is None else dy[:, pick].double().abs() * ~far
    wp, xd = w.detach()[pick].double(), x.detach().double()
    want, mag = dz @ wp, dz.abs() @ wp.abs()
    # products and sums of eleven terms in float32, one rounding to 8 bits
    assert ((dx.double() - want).abs() <= 2.0 ** -8 * want.abs() + 16 * F32 * mag + loose @ wp.abs() + 1e-30).all()
    want, mag = dz.t() @ xd, dz.abs().t() @ xd.abs()
    assert ((dw[pick].double() - want).abs() <= 2.0 ** -8 * want.abs() + (M + 4) * F32 * mag + loose.t() @ xd.abs() + 1e-30).all()
    assert not dw[5000].any() and not dw[N - 2].any()
