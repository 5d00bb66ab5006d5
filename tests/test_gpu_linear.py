"""linear against a plain implementation in 64 bits, forward and backward.

Tolerances, u the unit roundoff of the operands' type (2^-11, 2^-8): a product of
K terms in float32 is off by at most K 2^-24 of its terms' magnitudes; the
activations are within 2^-20 of their largest argument; y is rounded once. The
backward may round z (u |z|, times the slope's own slope, at most 1.13, in dy) and
dz (u |dz|) before its products, so dx and dw are off by those errors summed over
their terms' magnitudes, and rounded once; db is the sum of the unrounded dz. (Slopes
in steps of 2^-14 instead of a rounded z: 2^-15 of dy more.)
"""

from __future__ import annotations

import math

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_linear import ACTIVATIONS, _LinearFn

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}  # half a subnormal step
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def act(z, name):
    if name is None:
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)


def make(M, N, K, dtype, seed, bias=True, residual=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"x": r(M, K).to(dtype), "w": (r(N, K) / math.sqrt(K)).to(dtype), "b": (0.5 * r(N)).to(dtype) if bias else None,
            "r": r(M, N).to(dtype) if residual else None, "dy": r(M, N).to(dtype)}


def exact(s, name):
    """(outputs, tolerances) in 64 bits."""
    u, tiny = UNIT[s["x"].dtype], TINY[s["x"].dtype]
    x, w, dy = s["x"].double(), s["w"].double(), s["dy"].double()
    K, (M, N) = x.shape[1], dy.shape
    b = torch.zeros(N, dtype=torch.float64) if s["b"] is None else s["b"].double()
    z = x @ w.t() + b
    ze = F32 * (K + 4) * (x.abs() @ w.abs().t() + b.abs())
    a, slope = act(z, name)
    y = a if s["r"] is None else a + s["r"].double()
    ae = 1.13 * ze + 2.0 ** -20 * z.abs() + F32 * y.abs()
    if name is None:
        se = torch.zeros_like(z)
    else:  # z's rounding moves its slope; relu's jumps where z is within it of zero
        zr = ze + u * z.abs() + tiny
        se = (z.abs() <= zr).double() if name == "relu" else 1.13 * zr + 2.0 ** -20 * (1 + z.abs()) + 2.0 ** -15
    dz = dy * slope
    dze = dy.abs() * se
    dzr = dze + u * (dz.abs() + dze) + tiny  # of the products' operand
    return ({"y": y, "dx": dz @ w, "dw": dz.t() @ x, "db": dz.sum(0), "dr": dy},
            {"y": ae + u * (y.abs() + ae) + tiny,
             "dx": dzr @ w.abs() + F32 * (N + 4) * (dz.abs() @ w.abs()) + u * (dz @ w).abs() + tiny,
             "dw": dzr.t() @ x.abs() + F32 * (M + 4) * (dz.abs().t() @ x.abs()) + u * (dz.t() @ x).abs() + tiny,
             "db": dze.sum(0) + F32 * (M + 4) * dz.abs().sum(0) + u * dz.sum(0).abs() + tiny,
             "dr": torch.zeros_like(dy)})


def check(name, got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    off = (got - want).abs()
    ok = off <= tol * 1.01
    assert bool(ok.all()), f"{name}: {(~ok).sum().item()} off, by up to {off.max().item()}, {(off / tol).max().item()} of the tolerance"


def run(s, name, leaves=("x", "w", "b", "r")):
    t = {k: None if v is None else v.cuda() for k, v in s.items()}
    names = [k for k in leaves if t[k] is not None]
    for k in names:
        t[k].requires_grad_(True)
    y = fm.linear(t["x"], t["w"], t["b"], name, t["r"])
    grads = torch.autograd.grad(y, [t[k] for k in names], t["dy"])
    return {"y": y} | {"d" + k: g for k, g in zip(names, grads)}


def verify(s, name, leaves=("x", "w", "b", "r")):
    want, tol = exact(s, name)
    got = run(s, name, leaves)
    for k, v in got.items():
        check(k, v, want[k], tol[k])
    return got


# tiles are 64, 128 or 256 wide, stages 64 (32) deep, rows' groups 8: sizes around and off all of them
SIZES = [(1, 1, 1), (1, 8, 8), (2, 7, 9), (16, 16, 32), (31, 33, 65), (32, 128, 768), (64, 64, 64), (65, 63, 72),
         (127, 129, 130), (200, 77, 300), (257, 255, 256), (300, 520, 33), (513, 128, 2048), (1003, 77, 300), (1500, 9, 40)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_sizes(M, N, K, dtype):
    verify(make(M, N, K, dtype, M + N + K, residual=M % 2 == 0), ACTS[(M + N + K) % 5])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("bias,residual", [(True, True), (False, False)])
def test_activations(name, bias, residual, dtype):
    verify(make(130, 96, 80, dtype, 7, bias, residual), name)


@pytest.mark.parametrize("M,N,K", [(4200, 4104, 72), (5000, 2000, 264), (2100, 264, 1030), (100, 2056, 4200), (6000, 520, 520)])
def test_large_tiles_and_splits(M, N, K):
    """Every tile of the three products, and k split over workgroups."""
    verify(make(M, N, K, torch.bfloat16, 3, residual=True), "gelu")


@pytest.mark.parametrize("leaves", [("x",), ("w",), ("b",), ("r",), ("w", "b")])
def test_only_some_gradients(leaves):
    s = make(150, 72, 48, torch.float16, 11, residual=True)
    got = verify(s, "silu", leaves)
    assert set(got) == {"y"} | {"d" + k for k in leaves}


def test_views_and_leading_dims():
    s = make(24, 40, 48, torch.float16, 5, residual=True)
    want, tol = exact(s, "gelu")
    x, w, b, r, dy = (s[k].cuda() for k in ("x", "w", "b", "r", "dy"))
    wide = torch.full((24, 67), float("nan"), dtype=torch.float16, device="cuda")  # what lies beside is never used
    wide[:, 5:53] = x
    wpad = torch.full((40, 64), float("nan"), dtype=torch.float16, device="cuda")
    wpad[:, :48] = w
    rpad = torch.full((24, 43), float("nan"), dtype=torch.float16, device="cuda")
    rpad[:, 1:41] = r
    check("y", fm.linear(wide[:, 5:53], wpad[:, :48], b, "gelu", rpad[:, 1:41]), want["y"], tol["y"])
    check("y", fm.linear(x.t().contiguous().t(), w.t().contiguous().t(), b, "gelu", r.t().contiguous().t()), want["y"], tol["y"])
    y = fm.linear(x.view(2, 3, 4, 48), w, b, "gelu", r.view(2, 3, 4, 40))
    assert y.shape == (2, 3, 4, 40)
    check("y", y.view(24, 40), want["y"], tol["y"])
    xg, wg = x.view(4, 6, 48).requires_grad_(True), w.requires_grad_(True)
    y = fm.linear(xg, wg, b, "gelu", r.view(4, 6, 40))
    dx, dw = torch.autograd.grad(y, (xg, wg), dy.t().contiguous().t().view(4, 6, 40))
    check("dx", dx.view(24, 48), want["dx"], tol["dx"])
    check("dw", dw, want["dw"], tol["dw"])
    # a padded store whose K is no multiple of 8
    s = make(24, 40, 45, torch.float16, 6)
    want, tol = exact(s, None)
    wide = torch.full((24, 48), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, :45] = s["x"].cuda()
    check("y", fm.linear(wide[:, :45], s["w"].cuda(), s["b"].cuda()), want["y"], tol["y"])


def test_expanded_gradient_and_broadcast_input():
    s = make(30, 48, 64, torch.bfloat16, 8)
    s["dy"] = torch.ones(30, 48, dtype=torch.bfloat16)
    want, tol = exact(s, "silu")
    x, w, b = (s[k].cuda().requires_grad_(True) for k in ("x", "w", "b"))
    dx, dw, db = torch.autograd.grad(fm.linear(x, w, b, "silu").sum(), (x, w, b))
    for k, v in (("dx", dx), ("dw", dw), ("db", db)):
        check(k, v, want[k], tol[k])
    one = s["x"][:1].cuda().requires_grad_(True)  # a row read for every row
    y = fm.linear(one.expand(30, 64), w, b, "silu")
    (d1,) = torch.autograd.grad(y, one, s["dy"].cuda())
    t = {**s, "x": s["x"][:1].expand(30, 64)}
    want, tol = exact(t, "silu")
    check("y", y, want["y"], tol["y"])
    got = d1.cpu().double()[0]
    u = UNIT[torch.bfloat16]
    assert ((got - want["dx"].sum(0)).abs() <= tol["dx"].sum(0) + 30 * u * want["dx"].abs().sum(0)).all()


def test_no_rows():
    w = torch.ones(8, 16, device="cuda", dtype=torch.float16, requires_grad=True)
    b = torch.zeros(8, device="cuda", dtype=torch.float16, requires_grad=True)
    x = torch.empty(0, 16, device="cuda", dtype=torch.float16, requires_grad=True)
    y = fm.linear(x, w, b, "gelu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 8, device="cuda", dtype=torch.float16))
    assert y.shape == (0, 8) and dx.shape == (0, 16) and not dw.any() and not db.any()


@pytest.mark.parametrize("N,K", [(8192, 8192), (8200, 16379), (3, 5)])
def test_no_rows_of_a_large_weight(N, K):
    """64 threads an element would pass a launch's 2^32 from 2^26 elements on."""
    w = torch.ones(N, K, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    b = torch.ones(N, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    x = torch.empty(2, 0, K, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    torch.full((N * K + N,), float("nan"), device="cuda", dtype=torch.bfloat16)  # freed: what dw and db may get holds no zeros
    y = fm.linear(x, w, b, "silu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(2, 0, N, device="cuda", dtype=torch.bfloat16))
    assert y.shape == (2, 0, N) and dx.shape == x.shape and dw.shape == (N, K) and not dw.any() and not db.any()


def test_values_that_are_not_finite_stay_in_their_row():
    for M, N, K in ((70, 40, 48), (300, 200, 1000)):
        s = make(M, N, K, torch.float16, 2)
        s["x"][3, 5] = float("nan")
        s["x"][60, 0] = float("inf")
        for name in ACTS:
            y = fm.linear(s["x"].cuda(), s["w"].cuda(), s["b"].cuda(), name).cpu()
            bad = (~torch.isfinite(y)).any(1).nonzero().flatten().tolist()
            assert set(bad) <= {3, 60} and torch.isnan(y[3]).all()


@pytest.mark.parametrize("dtype,far", [(torch.float16, 200.0), (torch.bfloat16, 1e37)])
@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
def test_extreme_arguments(name, dtype, far):
    """Activations far out: the identity above, zero below, finite slopes."""
    x = torch.tensor([[-far], [-30.0], [-12.0], [-6.0], [0.0], [6.0], [12.0], [30.0], [far]], dtype=dtype)
    s = {"x": x, "w": torch.ones(1, 1, dtype=dtype), "b": None, "r": None, "dy": torch.ones(9, 1, dtype=dtype)}
    verify(s, name)


@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
def test_arguments_past_float16(name):
    """z beyond 65504 is infinite in float16; the slope there is still zero below and one above."""
    x = torch.tensor([[-300.0], [300.0]], dtype=torch.float16).cuda().requires_grad_(True)
    w = torch.full((1, 1), 300.0, dtype=torch.float16).cuda()
    y = fm.linear(x, w, None, name)
    (dx,) = torch.autograd.grad(y, x, torch.ones(2, 1, dtype=torch.float16).cuda())
    assert y[0].item() == 0 and math.isinf(y[1].item()) and dx[:, 0].tolist() == [0.0, 300.0]


def test_gradients_are_not_differentiable_again():
    s = make(20, 16, 24, torch.float16, 3)
    x, w = s["x"].cuda().requires_grad_(True), s["w"].cuda()
    for y in (fm.linear(x, w, None, "gelu"), fm.linear(x.t().contiguous().t(), w, None, "gelu"), fm.layer_norm(x)):
        (dx,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            dx.float().square().sum().backward()


@pytest.mark.parametrize("name", [None, "gelu", "gelu_tanh", "silu"])
def test_gradient_against_differences(name):
    s = make(40, 24, 32, torch.float16, 31, residual=True)
    got = run(s, name)
    args = {k: s[k].double() for k in ("x", "w", "b", "r")}

    def f(x, w, b, r):
        return ((act(x @ w.t() + b, name)[0] + r) * s["dy"].double()).sum()

    g = torch.Generator().manual_seed(2)
    for k in args:
        d = torch.randn(args[k].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, dn = (f(**{n: t + e * h * d if n == k else t for n, t in args.items()}) for e in (1, -1))
        mine = got["d" + k].cpu().double() * d
        # dz, z and the gradient rounded to 11 bits: three errors of 2^-11 of each term at most
        assert abs(mine.sum() - (up - dn) / (2 * h)) <= 4 * 2.0 ** -11 * 3 * mine.abs().sum(), k


def columns_first(t):
    return t.t().contiguous().t() if t.dim() == 2 else t.clone()


HOOKS = [(lambda t: t.cpu(), lambda t: t.cuda()), (lambda t: t, lambda t: t.contiguous().clone()), (lambda t: t, columns_first)]


@pytest.mark.parametrize("name", [None, "silu"])
@pytest.mark.parametrize("K", [96, 77])
@pytest.mark.parametrize("pack,unpack", HOOKS)
def test_saved_tensors_in_another_layout(pack, unpack, K, name):
    M, N = 150, 72
    s = {k: v.cuda() for k, v in make(M, N, K, torch.float16, 14, residual=True).items()}
    x = torch.zeros(M, 128, device="cuda", dtype=torch.float16)[:, :K].copy_(s["x"]).requires_grad_(True)
    w = torch.zeros(N, 256, device="cuda", dtype=torch.float16)[:, :K].copy_(s["w"]).requires_grad_(True)
    for fn in (fm.linear, lambda x, w, b, a, r: _LinearFn.apply(x, w, b, ACTIVATIONS[a], r)):
        want = torch.autograd.grad(fn(x, w, s["b"], name, s["r"]), (x, w), s["dy"])
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            y = fn(x, w, s["b"], name, s["r"])
        got = torch.autograd.grad(y, (x, w), s["dy"])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:-1]):
        y = fm.linear(x, w, s["b"], name, s["r"])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, (x, w), s["dy"])


def test_repeats_bit_for_bit_and_on_another_stream():
    s = make(3000, 200, 600, torch.bfloat16, 8, residual=True)
    a = run(s, "gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run(s, "gelu")
    side.synchronize()
    assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("M,N,K", [(64, 128, 2048), (700, 300, 256)])
def test_graph_replays(M, N, K):
    s = make(M, N, K, torch.float16, 12)
    x, w, b = (s[k].cuda() for k in ("x", "w", "b"))
    fm.linear(x, w, b, "silu")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fm.linear(x, w, b, "silu")
    for seed in range(3):
        x.copy_(make(M, N, K, torch.float16, 40 + seed)["x"])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, fm.linear(x, w, b, "silu"))


def test_refusals():
    x = torch.zeros(4, 16, device="cuda", dtype=torch.float16)
    w = torch.zeros(8, 16, device="cuda", dtype=torch.float16)
    b = torch.zeros(8, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError):
        fm.linear(x, w, b, "tanh")
    for bad in (dict(weight=w[:, :15]), dict(weight=w[0]), dict(bias=b[:7]), dict(residual=x)):
        with pytest.raises(AssertionError):
            fm.linear(**({"x": x, "weight": w, "bias": b} | bad))
    for bad in (dict(x=x.float()), dict(weight=w.bfloat16()), dict(bias=b.float()), dict(residual=torch.zeros(4, 8, device="cuda"))):
        with pytest.raises(TypeError):
            fm.linear(**({"x": x, "weight": w, "bias": b} | bad))
    with pytest.raises(TypeError):
        fm.linear(x.float(), w.float())
    with pytest.raises(RuntimeError):
        fm.linear(x.cpu(), w.cpu())
    with pytest.raises(RuntimeError):
        fm.linear(x, w.cpu())


def test_views_read_with_their_sign():
    s = {k: v.cuda() for k, v in make(30, 24, 40, torch.float16, 6, residual=True).items()}
    got, want = [], []
    for out, f in ((got, torch._neg_view), (want, lambda t: -t)):
        leaves = [f(s[k]).detach().requires_grad_(True) for k in ("x", "w", "b", "r")]
        y = fm.linear(leaves[0], leaves[1], leaves[2], "gelu", leaves[3])
        out += [y, *torch.autograd.grad(y, leaves, f(s["dy"]))]
        y = fm.linear(s["x"].requires_grad_(True), s["w"], None, "gelu")
        out += torch.autograd.grad(y, s["x"], f(s["dy"]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tangents_refused():
    x = torch.randn(4, 16, device="cuda", dtype=torch.float16)
    w = torch.randn(8, 16, device="cuda", dtype=torch.float16)
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(x, x)
        for f in (lambda: fm.linear(t, w), lambda: fm.linear(w, t), lambda: fm.layer_norm(t)):
            with pytest.raises(NotImplementedError):
                f()
        inside = fm.linear(x, w), fm.layer_norm(x)
        leaf = x.clone().requires_grad_(True)
        dy = torch.ones(4, 8, device="cuda", dtype=torch.float16)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(fm.linear(leaf, w), leaf, torch.autograd.forward_ad.make_dual(dy, dy))
    assert torch.equal(inside[0], fm.linear(x, w)) and torch.equal(inside[1], fm.layer_norm(x))
