"""gated_linear against a plain implementation in 64 bits, forward and backward.

Tolerances, u the unit roundoff of the operands' type (2^-11, 2^-8): a product of
K terms in float32 is off by at most K 2^-24 of its terms' magnitudes; the
activations are within 2^-20 of their largest argument, they and their slopes move by at most
1.13 of their argument; y is rounded once. The factors that the backward multiplies dy
with are coded: bfloat16 2^-10 of a factor from 2^-16 on, 2^-8 below, float16 2^-16. dg and du are
rounded (u) before their products, so the gradients are off by those errors summed over
their terms' magnitudes, and rounded once; bias gradients are sums of the unrounded ones.
"""

from __future__ import annotations

import math

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_gated import _GatedLinearFn
from flash_maxsim_amd.flash_maxsim_linear import ACTIVATIONS
from test_gpu_linear import ACTS, F32, HOOKS, TINY, UNIT, act, check

pytestmark = pytest.mark.gpu

LEAVES = ("x", "wg", "wu", "bg", "bu")
TYPES = [torch.float16, torch.bfloat16]


def make(M, N, K, dtype, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"x": r(M, K).to(dtype), "wg": (r(N, K) / math.sqrt(K)).to(dtype), "wu": (r(N, K) / math.sqrt(K)).to(dtype),
            "bg": (0.5 * r(N)).to(dtype) if bias else None, "bu": (0.5 * r(N)).to(dtype) if bias else None,
            "dy": r(M, N).to(dtype)}


def coded(f, dtype):
    """What the code of a factor is off by at most."""
    if dtype == torch.float16:
        return f.abs() * 2.0 ** -16
    return torch.where(f.abs() < 2.0 ** -16, 2.0 ** -8, 2.0 ** -10) * f.abs() + 2.0 ** -80


def exact(s, name):
    """(outputs, tolerances) in 64 bits."""
    dtype = s["x"].dtype
    u_, tiny = UNIT[dtype], TINY[dtype]
    x, wg, wu, dy = (s[k].double() for k in ("x", "wg", "wu", "dy"))
    K, (M, N) = x.shape[1], dy.shape
    bg, bu = (torch.zeros(N, dtype=torch.float64) if s[k] is None else s[k].double() for k in ("bg", "bu"))
    g, u = x @ wg.t() + bg, x @ wu.t() + bu
    ge = F32 * (K + 4) * (x.abs() @ wg.abs().t() + bg.abs())
    ue = F32 * (K + 4) * (x.abs() @ wu.abs().t() + bu.abs())
    a, slope = act(g, name)
    y = a * u
    ae = 1.13 * ge + 2.0 ** -20 * g.abs()
    ye = ae * u.abs() + (a.abs() + ae) * ue + 2 * F32 * y.abs()
    if name is None:
        se = torch.zeros_like(g)
    elif name == "relu":
        se = (g.abs() <= ge).double()
    else:
        se = 1.13 * ge + 2.0 ** -20 * (1 + g.abs())
    fg, fge = u * slope, (slope.abs() + se) * ue + u.abs() * se + F32 * (u * slope).abs()
    fge, fae = fge + coded(fg.abs() + fge, dtype), ae + coded(a.abs() + ae, dtype)
    dg, du = dy * fg, dy * a
    dge, due = dy.abs() * fge + F32 * dg.abs(), dy.abs() * fae + F32 * du.abs()
    rg, ru = dge + u_ * (dg.abs() + dge) + tiny, due + u_ * (du.abs() + due) + tiny  # of the products' operands
    dx, dwg, dwu = dg @ wg + du @ wu, dg.t() @ x, du.t() @ x
    return ({"y": y, "dx": dx, "dwg": dwg, "dwu": dwu, "dbg": dg.sum(0), "dbu": du.sum(0)},
            {"y": ye + u_ * (y.abs() + ye) + tiny,
             "dx": rg @ wg.abs() + ru @ wu.abs() + F32 * (2 * N + 4) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
             + u_ * dx.abs() + tiny,
             "dwg": rg.t() @ x.abs() + F32 * (M + 4) * (dg.abs().t() @ x.abs()) + u_ * dwg.abs() + tiny,
             "dwu": ru.t() @ x.abs() + F32 * (M + 4) * (du.abs().t() @ x.abs()) + u_ * dwu.abs() + tiny,
             "dbg": dge.sum(0) + F32 * (M + 4) * dg.abs().sum(0) + u_ * dg.sum(0).abs() + tiny,
             "dbu": due.sum(0) + F32 * (M + 4) * du.abs().sum(0) + u_ * du.sum(0).abs() + tiny})


def run(s, name, leaves=LEAVES):
    t = {k: None if v is None else v.cuda() for k, v in s.items()}
    names = [k for k in leaves if t[k] is not None]
    for k in names:
        t[k].requires_grad_(True)
    y = fm.gated_linear(*(t[k] for k in LEAVES), name)
    grads = torch.autograd.grad(y, [t[k] for k in names], t["dy"])
    return {"y": y} | {"d" + k: g for k, g in zip(names, grads)}


def verify(s, name, leaves=LEAVES):
    want, tol = exact(s, name)
    got = run(s, name, leaves)
    # float16 ends at 65504: what lies past 65520 rounds to infinity
    top = 65520.0 if s["x"].dtype == torch.float16 else math.inf
    for k, v in got.items():
        past = want[k].abs() - tol[k] > top
        over = torch.where(past, want[k].sign() * math.inf, 0.0)
        assert torch.equal(v.cpu().double()[past], over[past]), k
        check(k, torch.where(past.cuda(), 0.0, v.detach()), torch.where(past, 0.0, want[k]), tol[k])
    t = {k: None if s[k] is None else s[k].cuda() for k in LEAVES}
    assert torch.equal(fm.gated_linear(*t.values(), name), got["y"])  # without autograd
    return got


SIZES = [(1, 1, 1), (1, 8, 8), (2, 7, 9), (16, 16, 32), (17, 40, 264), (31, 33, 65), (32, 128, 768), (48, 24, 1000), (64, 64, 64),
         (65, 63, 72), (127, 129, 130), (200, 77, 300), (257, 255, 256), (300, 520, 33), (513, 128, 2048), (1003, 77, 300),
         (1500, 9, 40)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_sizes(M, N, K, dtype):
    verify(make(M, N, K, dtype, M + N + K, bias=M % 2 == 0), ACTS[(M + N + K) % 5])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("bias", [True, False])
def test_activations(name, bias, dtype):
    verify(make(130, 96, 80, dtype, 7, bias), name)
    verify(make(40, 96, 80, dtype, 8, bias), name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(4200, 2056, 72), (5000, 1000, 264), (2100, 136, 1030), (100, 2056, 2200), (6000, 264, 520)])
def test_large_tiles_and_splits(M, N, K, dtype):
    """Every tile of the three products, and k split over workgroups."""
    verify(make(M, N, K, dtype, 3), "gelu" if dtype == torch.float16 else "silu")


@pytest.mark.parametrize("leaves", [("x",), ("wg",), ("wu",), ("bg",), ("bu",), ("wu", "bg"), ("x", "bu")])
def test_only_some_gradients(leaves):
    got = verify(make(150, 72, 48, torch.float16, 11), "silu", leaves)
    assert set(got) == {"y"} | {"d" + k for k in leaves}


def test_one_bias():
    for k in ("bg", "bu"):
        s = make(70, 40, 48, torch.bfloat16, 12)
        s[k] = None
        verify(s, "gelu")


def test_views_and_leading_dims():
    s = make(24, 40, 48, torch.float16, 5)
    want, tol = exact(s, "gelu")
    t = {k: v.cuda() for k, v in s.items()}
    fused = torch.full((80, 64), float("nan"), dtype=torch.float16, device="cuda")  # what lies beside is never used
    fused[:40, :48], fused[40:, :48] = t["wg"], t["wu"]
    wide = torch.full((24, 67), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, 5:53] = t["x"]
    check("y", fm.gated_linear(wide[:, 5:53], fused[:40, :48], fused[40:, :48], t["bg"], t["bu"], "gelu"), want["y"], tol["y"])
    check("y", fm.gated_linear(t["x"].t().contiguous().t(), t["wg"].t().contiguous().t(), t["wu"], t["bg"], t["bu"], "gelu"),
          want["y"], tol["y"])
    # weights whose rows lie differently far apart, in both passes
    x, wg, wu = (v.detach().requires_grad_(True) for v in (t["x"].view(2, 3, 4, 48), fused[:40, :48], t["wu"]))
    y = fm.gated_linear(x, wg, wu, t["bg"], t["bu"], "gelu")
    assert y.shape == (2, 3, 4, 40)
    check("y", y.view(24, 40), want["y"], tol["y"])
    grads = torch.autograd.grad(y, (x, wg, wu), t["dy"].t().contiguous().t().view(2, 3, 4, 40))
    for k, v in zip(("dx", "dwg", "dwu"), grads):
        check(k, v.reshape(want[k].shape), want[k], tol[k])
    # one weight for both: its gradient is the sum
    w = t["wg"].clone().requires_grad_(True)
    (both,) = torch.autograd.grad(fm.gated_linear(t["x"], w, w, t["bg"], t["bu"], "gelu"), w, t["dy"])
    want, tol = exact({**s, "wu": s["wg"]}, "gelu")
    total = want["dwg"] + want["dwu"]
    check("dw", both, total, tol["dwg"] + tol["dwu"] + UNIT[torch.float16] * total.abs())


def test_expanded_gradient_and_broadcast_input():
    s = make(30, 48, 64, torch.bfloat16, 8)
    s["dy"] = torch.ones(30, 48, dtype=torch.bfloat16)
    want, tol = exact(s, "silu")
    t = {k: s[k].cuda().requires_grad_(True) for k in LEAVES}
    for k, v in zip(LEAVES, torch.autograd.grad(fm.gated_linear(*t.values()).sum(), t.values())):
        check("d" + k, v, want["d" + k], tol["d" + k])
    one = s["x"][:1].cuda().requires_grad_(True)  # a row read for every row
    y = fm.gated_linear(one.expand(30, 64), *list(t.values())[1:])
    (d1,) = torch.autograd.grad(y, one, s["dy"].cuda())
    want, tol = exact({**s, "x": s["x"][:1].expand(30, 64)}, "silu")
    check("y", y, want["y"], tol["y"])
    u = UNIT[torch.bfloat16]
    assert ((d1.cpu().double()[0] - want["dx"].sum(0)).abs() <= tol["dx"].sum(0) + 30 * u * want["dx"].abs().sum(0)).all()


def test_no_rows():
    wg, wu = (torch.ones(8, 16, device="cuda", dtype=torch.float16, requires_grad=True) for _ in range(2))
    b = torch.zeros(8, device="cuda", dtype=torch.float16, requires_grad=True)
    x = torch.empty(3, 0, 16, device="cuda", dtype=torch.float16, requires_grad=True)
    y = fm.gated_linear(x, wg, wu, b, None, "gelu")
    dx, *others = torch.autograd.grad(y, (x, wg, wu, b), torch.empty(3, 0, 8, device="cuda", dtype=torch.float16))
    assert y.shape == (3, 0, 8) and dx.shape == x.shape and not any(t.any() for t in others)


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite_stay_in_their_row(dtype):
    for M, N, K in ((30, 40, 48), (70, 40, 48), (300, 200, 1000)):
        s = make(M, N, K, dtype, 2)
        s["x"][3, 5] = float("nan")
        s["x"][20, 0] = float("inf")
        for name in ACTS:
            got = run(s, name, ("x",))
            for t in got.values():
                bad = (~torch.isfinite(t)).any(1).nonzero().flatten().tolist()
                assert set(bad) <= {3, 20} and not torch.isfinite(t[3]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
def test_arguments_far_out(name, dtype):
    """Factors that are tiny or large keep their gradients to the tolerance of their code."""
    x = torch.tensor([[-60.0], [-30.0], [-12.0], [-6.0], [-1.27846], [0.0], [6.0], [12.0], [200.0]], dtype=dtype)
    for up in (1.0, 1024.0, 2.0 ** -10):
        s = {"x": x, "wg": torch.ones(1, 1, dtype=dtype), "wu": torch.zeros(1, 1, dtype=dtype), "bg": None,
             "bu": torch.full((1,), up, dtype=dtype), "dy": torch.ones(9, 1, dtype=dtype)}
        verify(s, name)
        verify({**s, "x": x.repeat(9, 1), "dy": s["dy"].repeat(9, 1)}, name)


@pytest.mark.parametrize("exponent", [12, 15, 16, 17, 30, 33, 45, 60, 70])
def test_large_factors(exponent):
    """bfloat16 factors of 2^16 and more are off by 2^-8 at most, one of the roundings that u counts: products of
    a row of x has one element, so that the products are exact but for a rounding, whatever their size."""
    g = torch.Generator().manual_seed(exponent)
    M, N, K = 40, 24, 8
    one = torch.zeros(M, K)
    one[torch.arange(M), torch.arange(M) % K] = torch.rand(M, generator=g) + 1.0
    s = {"x": one.bfloat16(), "wg": (torch.rand(N, K, generator=g) + 0.5).bfloat16(),
         "wu": ((torch.rand(N, K, generator=g) - 0.5) * 2.0 ** exponent).bfloat16(), "bg": None, "bu": None,
         "dy": (torch.randn(M, N, generator=g) * 2.0 ** -exponent).bfloat16()}
    got = run(s, None)
    x, wg, wu, dy = (s[k].double() for k in ("x", "wg", "wu", "dy"))
    dg, du = dy * (x @ wu.t()), dy * (x @ wg.t())
    u_ = 2.0 ** -8  # of the code, of dg or du, and of the result; terms of float32 sums besides
    step = (1 + u_) ** 3 * (1 + F32 * 2 * M) - 1
    for k, terms in (("dwg", (dg.t().abs() @ x.abs(), dg.t() @ x)), ("dwu", (du.t().abs() @ x.abs(), du.t() @ x)),
                     ("dx", (dg.abs() @ wg.abs() + du.abs() @ wu.abs(), dg @ wg + du @ wu))):
        assert ((got[k].cpu().double() - terms[1]).abs() <= step * terms[0] + TINY[torch.bfloat16]).all(), k


def test_small_factors_reach_the_weights():
    """A unit whose arguments all lie at -20, where SiLU is -4e-8: its gradients are those of the formula."""
    M, K = 256, 16
    for dtype in TYPES:
        g = torch.Generator().manual_seed(9)
        x = torch.rand(M, K, generator=g).to(dtype)
        s = {"x": x, "wg": torch.zeros(8, K, dtype=dtype), "wu": torch.randn(8, K, generator=g).to(dtype),
             "bg": torch.full((8,), -20.0, dtype=dtype), "bu": None, "dy": torch.full((M, 8), 1024.0, dtype=dtype)}
        want, _ = exact(s, "silu")
        got = run(s, "silu")
        for k in ("dwg", "dwu", "dbg"):
            # coded to 2^-8 at worst, rounded twice; float16: dg and du, of 4e-5, to half a subnormal step as well
            tol = 2.5 * 2.0 ** -8 * want[k].abs().max() + TINY[dtype] * M
            assert (got[k].cpu().double() - want[k]).abs().max() <= tol, (k, dtype)


@pytest.mark.parametrize("name", [None, "gelu", "gelu_tanh", "silu"])
def test_gradient_against_differences(name):
    s = make(40, 24, 32, torch.float16, 31)
    got = run(s, name)
    args = {k: s[k].double() for k in LEAVES}

    def f(x, wg, wu, bg, bu):
        return (act(x @ wg.t() + bg, name)[0] * (x @ wu.t() + bu) * s["dy"].double()).sum()

    g = torch.Generator().manual_seed(2)
    for k in args:
        d = torch.randn(args[k].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, dn = (f(**{n: t + e * h * d if n == k else t for n, t in args.items()}) for e in (1, -1))
        mine = got["d" + k].cpu().double() * d
        # dg or du, the factor and the gradient rounded to 11 bits or finer: three errors of 2^-11 of each term at most
        assert abs(mine.sum() - (up - dn) / (2 * h)) <= 4 * 2.0 ** -11 * 3 * mine.abs().sum(), k


def both_ways():
    return (fm.gated_linear, lambda x, wg, wu, bg, bu, a: _GatedLinearFn.apply(x, wg, wu, bg, bu, ACTIVATIONS[a]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [96, 77])
@pytest.mark.parametrize("pack,unpack", HOOKS)
def test_saved_tensors_in_another_layout(pack, unpack, K, dtype):
    M, N = 150, 72
    s = {k: v.cuda() for k, v in make(M, N, K, dtype, 14).items()}
    x = torch.zeros(M, 128, device="cuda", dtype=dtype)[:, :K].copy_(s["x"]).requires_grad_(True)
    wg = torch.zeros(N, 256, device="cuda", dtype=dtype)[:, :K].copy_(s["wg"]).requires_grad_(True)
    leaves = (x, wg, s["wu"].requires_grad_(True))
    for fn in both_ways():
        want = torch.autograd.grad(fn(*leaves, s["bg"], s["bu"], "silu"), leaves, s["dy"])
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            y = fn(*leaves, s["bg"], s["bu"], "silu")
        got = torch.autograd.grad(y, leaves, s["dy"])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_both_paths_agree():
    s = {k: v.cuda() for k, v in make(300, 200, 136, torch.bfloat16, 21).items()}
    results = []
    for fn in both_ways():
        leaves = [s[k].detach().clone().requires_grad_(True) for k in LEAVES]
        y = fn(*leaves, "gelu")
        results.append([y, *torch.autograd.grad(y, leaves, s["dy"])])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_gradients_are_not_differentiable_again():
    s = make(20, 16, 24, torch.float16, 3)
    x, wg, wu = s["x"].cuda().requires_grad_(True), s["wg"].cuda(), s["wu"].cuda()
    for t in (x, x.t().contiguous().t()):
        (dx,) = torch.autograd.grad(fm.gated_linear(t, wg, wu).float().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            dx.float().square().sum().backward()


def test_backward_twice_and_changed_operands():
    s = {k: v.cuda() for k, v in make(90, 40, 48, torch.bfloat16, 13).items()}
    leaves = [s[k].requires_grad_(True) for k in LEAVES]
    y = fm.gated_linear(*leaves)
    first = torch.autograd.grad(y, leaves, s["dy"], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, leaves, s["dy"])))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, s["dy"])
    y = fm.gated_linear(*leaves)
    with torch.no_grad():
        leaves[1].add_(1)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, s["dy"])


def test_repeats_bit_for_bit_and_on_another_stream():
    s = make(3000, 200, 600, torch.bfloat16, 8)
    a = run(s, "gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run(s, "gelu")
    side.synchronize()
    assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("M,N,K", [(64, 128, 768), (100, 128, 2048), (700, 300, 256)])
def test_graph_replays(M, N, K):
    """Forward and backward in one graph, replayed with eager calls between."""
    s = make(M, N, K, torch.float16, 12)
    leaves = [s[k].cuda().requires_grad_(True) for k in LEAVES]
    dy = s["dy"].cuda()

    def step():
        y = fm.gated_linear(*leaves, "silu")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        with torch.no_grad():
            leaves[0].copy_(make(M, N, K, torch.float16, 40 + seed)["x"])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals():
    x = torch.zeros(4, 16, device="cuda", dtype=torch.float16)
    w = torch.zeros(8, 16, device="cuda", dtype=torch.float16)
    b = torch.zeros(8, device="cuda", dtype=torch.float16)
    good = {"x": x, "weight_gate": w, "weight_up": w, "bias_gate": b, "bias_up": b}
    with pytest.raises(ValueError):
        fm.gated_linear(**good, activation="tanh")
    for bad in (dict(weight_gate=w[:, :15]), dict(weight_up=w[:7]), dict(weight_gate=w[0]), dict(bias_gate=b[:7]),
                dict(bias_up=w), dict(x=x[:, :8])):
        with pytest.raises(AssertionError):
            fm.gated_linear(**(good | bad))
    for bad in (dict(x=x.float()), dict(weight_gate=w.bfloat16()), dict(bias_up=b.float())):
        with pytest.raises(TypeError):
            fm.gated_linear(**(good | bad))
    with pytest.raises(TypeError):
        fm.gated_linear(x.float(), w.float(), w.float())
    for bad in (dict(x=x.cpu()), dict(weight_up=w.cpu()), dict(bias_gate=b.cpu())):
        with pytest.raises(RuntimeError):
            fm.gated_linear(**(good | bad))


def test_views_read_with_their_sign():
    s = {k: v.cuda() for k, v in make(30, 24, 40, torch.float16, 6).items()}
    got, want = [], []
    for out, f in ((got, torch._neg_view), (want, lambda t: -t)):
        leaves = [f(s[k]).detach().requires_grad_(True) for k in LEAVES]
        y = fm.gated_linear(*leaves, "gelu")
        out += [y, *torch.autograd.grad(y, leaves, f(s["dy"]))]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tangents_refused():
    x = torch.randn(4, 16, device="cuda", dtype=torch.float16)
    w = torch.randn(8, 16, device="cuda", dtype=torch.float16)
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(x, x)
        u = torch.autograd.forward_ad.make_dual(w, w)
        for f in (lambda: fm.gated_linear(t, w, w), lambda: fm.gated_linear(x, u, w), lambda: fm.gated_linear(x, w, u)):
            with pytest.raises(NotImplementedError):
                f()
        inside = fm.gated_linear(x, w, w)
    assert torch.equal(inside, fm.gated_linear(x, w, w))
