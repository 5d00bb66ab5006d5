"""The encoder block's operators past 2^32 elements, where 32-bit offsets would wrap."""

from __future__ import annotations

import pytest
import torch

import flash_maxsim_amd as fm
from test_gpu_layers_large import filled

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
U16 = 2.0 ** -11
DEV = "cuda"


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB of free GPU memory")
    yield
    torch.cuda.empty_cache()


def test_gated_linear():
    """y, the factors' planes, dg and du hold more than 2^32 elements each; the tiles go in several launches."""
    M, N, K = (1 << 22) + 333, 1032, 24
    x, part = filled(M, K, 1)
    g = torch.Generator(device=DEV).manual_seed(2)
    wg, wu = ((torch.randn(N, K, generator=g, device=DEV) / 5).half().requires_grad_(True) for _ in range(2))
    x.requires_grad_(True)
    y = fm.gated_linear(x, wg, wu, activation="silu")
    pick = torch.tensor([0, 1, 4099, 1 << 20, (1 << 22) - 1, 1 << 22, M - 200, M - 2, M - 1], device=DEV)
    rows, G, W = part[pick % 4099].double(), wg.detach().double(), wu.detach().double()
    a, u = rows @ G.t(), rows @ W.t()
    s = torch.sigmoid(a)
    ze = F32 * (K + 4) * (rows.abs() @ torch.maximum(G.abs(), W.abs()).t())
    ae = 1.13 * ze + 2.0 ** -20 * a.abs()
    assert ((y.detach()[pick].double() - a * s * u).abs() <= U16 * (a * s * u).abs() + ae * (u.abs() + ze) + (a * s).abs() * ze + 2.0 ** -24).all()
    dy = torch.zeros(M, N, dtype=torch.float16, device=DEV)
    dy[pick] = torch.randn(len(pick), N, generator=g, device=DEV).half()
    dx, dwg, dwu = torch.autograd.grad(y, (x, wg, wu), dy)
    d = dy[pick].double()
    dg, du = d * u * s * (1 + a * (1 - s)), d * a * s
    # each rounded to 11 bits, its factor coded to 16, and both off by the sums' errors with slopes below 1.13
    eg = U16 * dg.abs() + d.abs() * (2.0 ** -15 * (u * s).abs() + ze * 1.2 * (1 + u.abs()) + 2.0 ** -19 * u.abs()) + 2.0 ** -25
    eu = U16 * du.abs() + d.abs() * (2.0 ** -15 * (a * s).abs() + ae) + 2.0 ** -25
    want = dg @ G + du @ W
    assert ((dx[pick].double() - want).abs() <= 1.1 * (eg @ G.abs() + eu @ W.abs()) + 2 * U16 * want.abs() + 2.0 ** -20).all()
    assert not dx[5000].any() and not dx[M - 3].any()
    for got, z, e in ((dwg, dg, eg), (dwu, du, eu)):
        want = z.t() @ rows
        assert ((got.double() - want).abs() <= 1.1 * e.t() @ rows.abs() + 2 * U16 * want.abs() + 2.0 ** -20).all()


def test_residual_norm():
    M, d = (1 << 22) + 333, 1032
    x, part = filled(M, d, 3)
    g = torch.Generator(device=DEV).manual_seed(4)
    w = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).half().requires_grad_(True)
    x.requires_grad_(True)
    h, y = fm.residual_norm(x, x.detach(), w, norm="rms", post_norm=True)
    pick = torch.tensor([0, 4099, 1 << 21, (1 << 22) - 1, 1 << 22, M - 2, M - 1], device=DEV)
    small = part[pick % 4099].requires_grad_(True)
    w2 = w.detach().clone().requires_grad_(True)
    # rows are alike wherever they lie: those of a call of their own
    h2, y2 = fm.residual_norm(small, small.detach(), w2, norm="rms", post_norm=True)
    assert torch.equal(h[pick], h2) and torch.equal(y[pick], y2)
    v = part[(M - 1) % 4099].detach().double()
    v = v + v / torch.sqrt((v * v).mean() + 1e-5)
    assert ((h[M - 1].double() - v).abs() <= U16 * v.abs() + 1e-5).all()
    dy = torch.zeros(M, d, dtype=torch.float16, device=DEV)
    dy[pick] = torch.randn(len(pick), d, generator=g, device=DEV).half()
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    dx2, dw2 = torch.autograd.grad(y2, (small, w2), dy[pick])
    assert torch.equal(dx[pick], dx2) and not dx[5000].any() and not dx[M - 3].any()
    # the same seven terms of each column, in another order
    assert (dw.float() - dw2.float()).abs().max() <= 2 * U16 * dw2.abs().max()


def test_embedding():
    V, d, T = (1 << 22) + 333, 1032, 20000
    w, part = filled(V, d, 5)
    w.requires_grad_(True)
    g = torch.Generator(device=DEV).manual_seed(6)
    ids = torch.randint(V - 3000, V, (T,), generator=g, device=DEV)
    ids[:50] = torch.arange(50, device=DEV)
    y = fm.embedding(ids, w)
    assert torch.equal(y.detach(), part[ids % 4099])
    dy = torch.randn(T, d, generator=g, device=DEV).half()
    (dw,) = torch.autograd.grad(y, w, dy)
    want = torch.zeros(3000, d, dtype=torch.float64, device=DEV).index_add_(0, ids[50:] - (V - 3000), dy[50:].double())
    size = torch.zeros(3000, d, dtype=torch.float64, device=DEV).index_add_(0, ids[50:] - (V - 3000), dy[50:].double().abs())
    assert ((dw[V - 3000:].double() - want).abs() <= U16 * want.abs() + 64 * F32 * size + 2.0 ** -25).all()
    assert torch.equal(dw[:50], dy[:50]) and not any(t.any() for t in dw[50:V - 3000].split(1 << 20))


@pytest.mark.parametrize("T", [9, 5000, 40000])
@pytest.mark.parametrize("d,dtype", [(601, torch.float16), (299, torch.float32), (608, torch.bfloat16)])
def test_embedding_gradient_past_the_caches(T, d, dtype):
    """Tables whose gradient is stored past the caches, rows at any element."""
    V = 200003
    g = torch.Generator(device=DEV).manual_seed(T + d)
    ids = torch.randint(V - 20000, V, (T,), generator=g, device=DEV)
    ids[: T // 3] = 7
    w = torch.empty(V, d, device=DEV, dtype=dtype).requires_grad_(True)
    dy = torch.randn(T, d, generator=g, device=DEV).to(dtype)
    (dw,) = torch.autograd.grad(fm.embedding(ids, w), w, dy)
    want = torch.zeros(V, d, dtype=torch.float64, device=DEV).index_add_(0, ids, dy.double())
    size = torch.zeros(V, d, dtype=torch.float64, device=DEV).index_add_(0, ids, dy.double().abs())
    # the result's rounding, and float32 sums of fewer than T terms
    u = torch.finfo(dtype).eps / 2
    assert ((dw.double() - want).abs() <= u * want.abs() + F32 * T * size + 2.0 ** -25).all()


def test_embedding_of_many_tokens():
    """T x d past 2^32: rows of dy and of y."""
    T, V, d = (1 << 22) + 333, 500, 1032
    g = torch.Generator(device=DEV).manual_seed(7)
    dy, part = filled(T, d, 8)
    ids = torch.randint(0, V, (T,), generator=g, device=DEV)
    w = torch.randn(V, d, generator=g, device=DEV).half().requires_grad_(True)
    y = fm.embedding(ids, w, 0.5)
    for a in (0, 1 << 21, T - 1000):
        assert torch.equal(y.detach()[a:a + 1000], w.detach()[ids[a:a + 1000]] * 0.5)
    (dw,) = torch.autograd.grad(y, w, dy)
    rows = torch.arange(T, device=DEV) % 4099
    count = torch.zeros(V, 4099, dtype=torch.float64, device=DEV)
    count.index_put_((ids, rows), torch.ones((), dtype=torch.float64, device=DEV), accumulate=True)
    want = count @ part.double() * 0.5
    n = torch.bincount(ids, minlength=V).max().item()
    # a float32 sum of stretches of at most 32 terms, every sixteenth of them and the sixteen
    tol = F32 * (32 + n / 32 / 16 + 20) * (count @ part.double().abs()) * 0.5
    assert ((dw.double() - want).abs() <= U16 * want.abs() + tol + 2.0 ** -25).all()


def test_orthogonalize():
    """A matrix whose last rows and columns alone are not zero: the result there is the small matrix's, zeros elsewhere."""
    for rows, cols in ((4104, 1 << 20), ((1 << 20) - 24, 4104)):
        u = torch.zeros(rows, cols, device=DEV, dtype=torch.bfloat16)
        small = torch.randn(100, 300, generator=torch.Generator(device=DEV).manual_seed(9), device=DEV).bfloat16()
        u[-100:, -300:] = small
        got = fm.orthogonalize(u, steps=2)
        want = fm.orthogonalize(small.float(), steps=2)
        assert (got[-100:, -300:].float() - want).norm() <= 2.0 ** -8 * want.norm()
        assert not got[:-100].any() and not got[-100:, :-300].any()
        del u, got
