"""layer_norm against a plain implementation in 64 bits, forward and backward.

Tolerances: an output in a type of unit roundoff u is rounded once, u |exact|; its
float32 sums of d terms run over lanes of at most d / 64 + 1 terms (a workgroup's
rows fewer) and a tree of 9, so each sum is off by at most (d / 64 + 10) 2^-24 of
its terms' magnitudes, and a handful of products and a root add 2^-24 each. The
weight's gradient sums M rows the same way, at most M terms one by one.
"""

from __future__ import annotations

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_norm import _LayerNormFn

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: F32}
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def make(M, d, dtype, seed, wdtype=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, d, generator=g) * (1 + torch.rand(M, 1, generator=g)) + torch.randn(M, 1, generator=g)).to(dtype)
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(wdtype or dtype)
    b = (0.2 * torch.randn(d, generator=g)).to(wdtype or dtype)
    dy = torch.randn(M, d, generator=g).to(dtype)
    return x, w, b, dy


def exact(x, w, b, dy, eps=1e-5):
    """(outputs, their float32 error in units of 2^-24) in 64 bits."""
    d = x.shape[1]
    x, dy = x.double(), dy.double()
    w = torch.ones(d, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(d, dtype=torch.float64) if b is None else b.double()
    K = d / 64 + 40
    mu = x.mean(1, keepdim=True)
    e = x - mu
    rs = 1 / torch.sqrt((e * e).mean(1, keepdim=True) + eps)
    xh = e * rs
    xerr = rs * (x.abs() + x.abs().mean(1, keepdim=True)) + xh.abs()  # of xh, in units of K 2^-24
    wdy = w * dy
    c1, c2 = wdy.mean(1, keepdim=True), (wdy * xh).mean(1, keepdim=True)
    a1, a2 = wdy.abs().mean(1, keepdim=True), (wdy.abs() * (xh.abs() + xerr)).mean(1, keepdim=True)
    out = {"y": xh * w + b, "dx": rs * (wdy - c1 - xh * c2), "dw": (dy * xh).sum(0), "db": dy.sum(0)}
    M = x.shape[0]
    err = {"y": K * (xerr * w.abs() + b.abs()),
           "dx": K * rs * (wdy.abs() + a1 + (xh.abs() + xerr) * a2 + xerr * c2.abs()),
           "dw": K * (dy.abs() * (xerr + xh.abs())).sum(0) + M * (dy * xh).abs().sum(0),
           "db": M * dy.abs().sum(0)}
    return out, err


def check(name, got, want, err):
    got = got.detach().cpu()
    u = UNIT[got.dtype]
    tol = u * want.abs() + F32 * err + (2.0 ** -25 if got.dtype == torch.float16 else 1e-38)
    off = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((off <= tol).all()), f"{name}: off by {off.max().item()}, {(off / tol).max().item()} of the tolerance"


def run(x, w, b, dy, eps=1e-5, **kw):
    leaves = [None if t is None else t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = fm.layer_norm(*leaves, eps=eps, **kw)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.cuda())
    names = [n for n, t in zip(("dx", "dw", "db"), leaves) if t is not None]
    return {"y": y} | dict(zip(names, grads))


WIDTHS = [1, 2, 7, 8, 63, 64, 65, 256, 300, 771, 1024, 1025, 1032, 2048, 2050, 4096, 5001, 8192, 8200, 16384, 16392]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_widths(d, dtype):
    M = 37 if d < 4096 else 5
    x, w, b, dy = make(M, d, dtype, d)
    want, err = exact(x, w, b, dy)
    for k, v in run(x, w, b, dy).items():
        check(k, v, want[k], err[k])
    y = fm.layer_norm(x.cuda(), w.cuda(), b.cuda())  # without the backward's statistics
    check("y alone", y, want["y"], err["y"])


@pytest.mark.parametrize("M", [1, 2, 9, 1000, 5003])
@pytest.mark.parametrize("d", [128, 130, 1536, 9000])
def test_rows(M, d):
    if M * d > 10_000_000:
        M = 700
    x, w, b, dy = make(M, d, torch.bfloat16, M)
    want, err = exact(x, w, b, dy)
    for k, v in run(x, w, b, dy).items():
        check(k, v, want[k], err[k])


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
def test_optional_and_mixed_weights(which, wdtype):
    x, w, b, dy = make(50, 200, torch.bfloat16, 3, wdtype)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    want, err = exact(x, w, b, dy)
    got = run(x, w, b, dy)
    for k, v in got.items():
        check(k, v, want[k], err[k])
    for k in ("dw", "db"):
        assert k not in got or got[k].dtype == wdtype


def test_views_and_leading_dims():
    x, w, b, dy = make(24, 96, torch.float16, 5)
    want, err = exact(x, w, b, dy)
    wide = torch.zeros(24, 133, dtype=torch.float16, device="cuda")
    wide[:, 3:99] = x.cuda()  # rows off every alignment
    check("y", fm.layer_norm(wide[:, 3:99], w.cuda(), b.cuda()), want["y"], err["y"])
    check("y", fm.layer_norm(x.cuda().t().contiguous().t(), w.cuda(), b.cuda()), want["y"], err["y"])
    y = fm.layer_norm(x.cuda().view(2, 3, 4, 96), w.cuda(), b.cuda())
    assert y.shape == (2, 3, 4, 96)
    check("y", y.view(24, 96), want["y"], err["y"])
    xg = x.cuda().view(4, 6, 96).requires_grad_(True)
    (dx,) = torch.autograd.grad(fm.layer_norm(xg, w.cuda(), b.cuda()), xg, dy.cuda().view(4, 6, 96))
    check("dx", dx.view(24, 96), want["dx"], err["dx"])
    # the gradient of a sum is expanded, and one row is broadcast to many
    one = x[:1].cuda().requires_grad_(True)
    (dx,) = torch.autograd.grad(fm.layer_norm(one.expand(24, 96), w.cuda(), b.cuda()).sum(), one)
    w1, e1 = exact(x[:1], w, b, torch.ones(1, 96))
    got = dx.detach().cpu().double()
    assert bool(((got - 24 * w1["dx"]).abs() <= 24 * (2 * 2.0 ** -11 * w1["dx"].abs() + F32 * e1["dx"] + 2.0 ** -24)).all())


def test_no_rows_and_constant_rows():
    w = torch.ones(64, device="cuda", requires_grad=True)
    b = torch.zeros(64, device="cuda", requires_grad=True)
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    y = fm.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 64, device="cuda"))
    assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()
    # a row of equal values has no deviation: y is the bias, and nothing is not finite
    x = torch.full((3, 64), 5.0, device="cuda", requires_grad=True)
    y = fm.layer_norm(x, w, b)
    (dx,) = torch.autograd.grad(y, x, torch.ones(3, 64, device="cuda"))
    assert not y.any() and torch.isfinite(dx).all()


def test_large_mean_keeps_its_digits():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(16, 512, generator=g) + 1000.0
    want, _ = exact(x, None, None, torch.zeros(16, 512))
    got = fm.layer_norm(x.cuda()).cpu().double()
    # the mean of values near 1000 is off by up to 18 * 2^-24 * 1000
    assert (got - want["y"]).abs().max() <= 2 * 18 * F32 * 1000 + 64 * F32


def test_rows_that_are_not_finite_stay_alone():
    x, w, b, dy = make(20, 100, torch.float32, 9)
    x[3, 5], x[7, 1] = float("nan"), float("inf")
    y = fm.layer_norm(x.cuda(), w.cuda(), b.cuda()).cpu()
    bad = ~torch.isfinite(y).all(1)
    assert bad.nonzero().flatten().tolist() == [3, 7] and torch.isnan(y[3]).all()


@pytest.mark.parametrize("d", [40, 1500])
def test_gradient_against_differences(d):
    x, w, b, dy = make(3, d, torch.float32, 21)
    got = run(x, w, b, dy)

    def f(x, w, b):
        e = x - x.mean(1, keepdim=True)
        return ((e / torch.sqrt((e * e).mean(1, keepdim=True) + 1e-5) * w + b) * dy.double()).sum()

    args = [t.double() for t in (x, w, b)]
    h = 1e-5
    g = torch.Generator().manual_seed(2)
    for i, k in enumerate(("dx", "dw", "db")):
        u = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        plus, minus = (f(*[t + s * h * u if j == i else t for j, t in enumerate(args)]) for s in (1, -1))
        slope = (plus - minus) / (2 * h)
        mine = (got[k].cpu().double() * u).sum()
        scale = (got[k].cpu().double() * u).abs().sum()
        assert abs(mine - slope) <= 1e-5 * scale, k


def test_repeats_bit_for_bit_and_on_another_stream():
    x, w, b, dy = make(3000, 768, torch.bfloat16, 8)
    a = run(x, w, b, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = run(x, w, b, dy)
    side.synchronize()
    assert all(torch.equal(a[k], c[k]) for k in a)


def test_graph_replays():
    x, w, b, dy = make(300, 384, torch.float16, 12)
    xs, ws, bs, gs = (t.cuda() for t in (x, w, b, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fm.layer_norm(xs, ws, bs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fm.layer_norm(xs, ws, bs)
    for seed in range(3):
        xs.copy_(make(300, 384, torch.float16, 40 + seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, fm.layer_norm(xs, ws, bs))


def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    with pytest.raises(AssertionError):
        fm.layer_norm(x, torch.ones(7, device="cuda"))
    with pytest.raises(AssertionError):
        fm.layer_norm(torch.zeros(4, 0, device="cuda"))
    with pytest.raises(TypeError):
        fm.layer_norm(x.double())
    with pytest.raises(TypeError):
        fm.layer_norm(x.half(), torch.ones(8, device="cuda").bfloat16())
    with pytest.raises(TypeError):
        fm.layer_norm(x.half(), torch.ones(8, device="cuda"), torch.ones(8, device="cuda").half())
    with pytest.raises(RuntimeError):
        fm.layer_norm(x.cpu())
    with pytest.raises(RuntimeError):
        fm.layer_norm(x, torch.ones(8))
    with pytest.raises(RuntimeError, match="eps"):
        fm.layer_norm(x, eps=-1.0)
    with pytest.raises(RuntimeError, match="FMX_MAX_D"):
        fm.layer_norm(torch.zeros(1, 65537, device="cuda"))


@pytest.mark.parametrize("pack,unpack", [(lambda t: t.cpu(), lambda t: t.cuda()), (lambda t: t, lambda t: t.contiguous().clone()),
                                         (lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone())])
def test_saved_tensors_in_another_layout(pack, unpack):
    g = torch.Generator().manual_seed(3)
    x = torch.zeros(70, 512, device="cuda")[:, :300].copy_(torch.randn(70, 300, generator=g)).requires_grad_(True)
    w, b = (torch.randn(300, generator=g).cuda().requires_grad_(True) for _ in range(2))
    dy = torch.randn(70, 300, generator=g).cuda()
    for fn in (fm.layer_norm, lambda *a: _LayerNormFn.apply(*a, 1e-5)):
        want = torch.autograd.grad(fn(x, w, b), (x, w, b), dy)
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            y = fn(x, w, b)
        # the rows' alignment may differ, and with it the order of their sums: dw and db are sums of 70 rows
        for a, e in zip(torch.autograd.grad(y, (x, w, b), dy), want):
            assert (a - e).abs().max() <= 2.0 ** -24 * 300 * 8 * e.abs().max()


def test_views_read_with_their_sign():
    """The imaginary part of a conjugate is a view whose elements are stored negated."""
    g = torch.Generator().manual_seed(4)
    z = torch.complex(torch.randn(20, 33, generator=g), torch.randn(20, 33, generator=g)).cuda()
    w = torch._neg_view(torch.randn(33, generator=g).cuda())
    x, dy = z.conj().imag, torch._neg_view(torch.randn(20, 33, generator=g).cuda())
    assert x.is_neg() and w.is_neg() and dy.is_neg()
    got, want = ([fm.layer_norm(a, b)] + list(torch.autograd.grad(fm.layer_norm(a, b), (a, b), e)) for a, b, e in (
        [t.detach().requires_grad_(True) for t in (x, w)] + [dy],
        [t.detach().resolve_neg().contiguous().requires_grad_(True) for t in (x, w)] + [dy.resolve_neg()]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
