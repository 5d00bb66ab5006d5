"""residual_norm against a plain implementation in 64 bits, forward and backward.

Tolerances: an output in a type of unit roundoff u is rounded once, u |exact|. Everything before is float32: a sum of d
terms runs over lanes of at most d / 64 + 1 terms and a tree of 12, and a handful of products and roots follow
each other, so with K = d / 64 + 60 a value is off by at most K 2^-24 of the magnitudes that it is made of. `exact`
carries these magnitudes along beside every value (an inverse deviation moves with its row's errors by their
root mean square times itself). Sums over M rows add M 2^-24 of their terms' magnitudes.
"""

from __future__ import annotations

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_residual_norm import _ResidualNormFn

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: F32}
TYPES = list(UNIT)
ROWS = ("x", "r", "gate")
VECTORS = ("w", "b", "pw", "pb", "scale")
ALL = ("post", "gate", "scale")


def make(M, d, dtype, seed, parts=ALL, norm="layer", alpha=1.0, wdtype=None, bias=True):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    wt = wdtype or dtype
    s = {"x": (n(M, d) * (0.5 + torch.rand(M, 1, generator=g)) + n(M, 1)).to(dtype), "r": (n(M, d) + 0.5 * n(M, 1)).to(dtype),
         "gate": n(M, d).to(dtype) if "gate" in parts else None, "w": (1 + 0.2 * n(d)).to(wt),
         "b": (0.2 * n(d)).to(wt) if bias else None, "pw": (1 + 0.2 * n(d)).to(wt) if "post" in parts else None,
         "pb": (0.2 * n(d)).to(wt) if "post" in parts and bias else None,
         "scale": (0.5 + 0.2 * n(d)).to(wt) if "scale" in parts else None, "dh": n(M, d).to(dtype), "dy": n(M, d).to(dtype),
         "post": "post" in parts, "norm": norm, "alpha": alpha}
    return s


def mean(t):
    return t.mean(1, keepdim=True)


def normalised(v, e, norm, eps):
    """norm(v), the inverse deviation and the magnitudes of the result's errors and of the deviation's, from v's."""
    mu = mean(v) if norm == "layer" else torch.zeros_like(v[:, :1])
    c = v - mu
    rs = 1 / torch.sqrt(mean(c * c) + eps)
    xh = c * rs
    ce = e + (mean(v.abs() + e) + v.abs() if norm == "layer" else 0)
    re = 1 + rs * torch.sqrt(mean(ce * ce))  # relative, of rs
    return xh, rs, rs * ce + xh.abs() * re, re


def grad_of_norm(q, qe, xh, xe, rs, re, norm):
    """The gradient of norm(v) from xh's q, and the magnitudes of its errors."""
    c1, c2 = mean(q) if norm == "layer" else 0, mean(q * xh)
    a1 = mean(q.abs() + qe) if norm == "layer" else 0
    a2 = mean((q.abs() + qe) * (xh.abs() + xe))
    out = rs * (q - c1 - xh * c2)
    return out, rs * (q.abs() + qe + a1 + (xh.abs() + xe) * a2 * 2 + xe * c2.abs()) + out.abs() * re


def exact(s, eps=1e-5):
    """(outputs, magnitudes of their errors in units of K 2^-24) in 64 bits."""
    M, d = s["x"].shape
    norm, alpha = s["norm"], s["alpha"]
    D = {k: s[k].double() if s[k] is not None else None for k in ROWS + VECTORS + ("dh", "dy")}
    one = torch.ones(d, dtype=torch.float64)
    w, pw, scale = (one if D[k] is None else D[k] for k in ("w", "pw", "scale"))
    b, pb = (0 * one if D[k] is None else D[k] for k in ("b", "pb"))
    gate = torch.ones(M, d, dtype=torch.float64) if D["gate"] is None else D["gate"]
    t, te = D["x"], torch.zeros(M, d, dtype=torch.float64)
    if s["post"]:
        xh, rs1, xe, re1 = normalised(t, te, norm, eps)
        t = xh * pw + pb
        te = xe * pw.abs() + t.abs() + pb.abs()
    k = scale * gate
    h = alpha * D["r"] + k * t
    he = (alpha * D["r"]).abs() + k.abs() * (te + t.abs())
    hh, rs2, hhe, re2 = normalised(h, he, norm, eps)
    dy = torch.zeros_like(h) if D["dy"] is None else D["dy"]
    dh = torch.zeros_like(h) if D["dh"] is None else D["dh"]
    gn, gne = grad_of_norm(dy * w, (dy * w).abs(), hh, hhe, rs2, re2, norm)
    g, ge = dh + gn, dh.abs() + gne
    q, qe = g * k, (ge + g.abs()) * k.abs()
    out = {"h": h, "y": hh * w + b, "dr": alpha * g, "dgate": g * scale * t, "dw": (dy * hh).sum(0), "db": dy.sum(0),
           "dscale": (g * gate * t).sum(0)}
    err = {"h": he, "y": hhe * w.abs() + b.abs() + (hh * w).abs(), "dr": abs(alpha) * ge,
           "dgate": scale.abs() * (ge * t.abs() + g.abs() * te + (g * t).abs()),
           "dw": (dy.abs() * hhe).sum(0), "db": 0 * one, "dscale": (gate.abs() * (ge * t.abs() + g.abs() * te)).sum(0)}
    many = {"dw": (dy * hh).abs().sum(0), "db": dy.abs().sum(0), "dscale": (g * gate * t).abs().sum(0)}
    if s["post"]:
        out["dx"], err["dx"] = grad_of_norm(q * pw, qe * pw.abs(), xh, xe, rs1, re1, norm)
        out |= {"dpw": (q * xh).sum(0), "dpb": q.sum(0)}
        err |= {"dpw": (qe * xh.abs() + q.abs() * xe).sum(0), "dpb": qe.sum(0)}
        many |= {"dpw": (q * xh).abs().sum(0), "dpb": q.abs().sum(0)}
    else:
        out["dx"], err["dx"] = q, qe
    K = d / 64 + 60
    return out, {n: F32 * (K * e + M * many.get(n, 0)) for n, e in err.items()}


def check(name, got, want, err):
    got = got.detach().cpu()
    u = UNIT[got.dtype]
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    tol = u * (want.abs() + err) + err + tiny
    off = (got.double() - want).abs()
    assert got.shape == want.shape
    assert (off <= tol * 1.01).all(), f"{name}: off by up to {off.max().item()}, {(off / tol).max().item()} of the tolerance"


def call(t, s, fn=None, **kw):
    if fn is None:
        return fm.residual_norm(t["x"], t["r"], t["w"], t["b"], norm=s["norm"], post_norm=s["post"], post_weight=t["pw"],
                                post_bias=t["pb"], gate=t["gate"], scale=t["scale"], residual_scale=s["alpha"], **kw)
    return fn(*(t[k] for k in ROWS + VECTORS), s["post"], s["alpha"], int(s["norm"] == "rms"), 1e-5)


def run(s, leaves=ROWS + VECTORS, outputs=("h", "y"), fn=None):
    t = {k: None if s[k] is None else s[k].cuda() for k in ROWS + VECTORS + ("dh", "dy")}
    names = [k for k in leaves if t[k] is not None]
    for k in names:
        t[k].requires_grad_(True)
    h, y = call(t, s, fn)
    outs = [o for n, o in (("h", h), ("y", y)) if n in outputs]
    given = [t["d" + n] for n in ("h", "y") if n in outputs]
    grads = torch.autograd.grad(outs, [t[k] for k in names], given, allow_unused=True)
    return {"h": h, "y": y} | {"d" + k: g for k, g in zip(names, grads)}


def verify(s, leaves=ROWS + VECTORS):
    want, err = exact(s)
    got = run(s, leaves)
    for k, v in got.items():
        check(k, v, want[k], err[k])
    t = {k: None if s[k] is None else s[k].cuda() for k in ROWS + VECTORS}
    h, y = call(t, s)
    assert torch.equal(h, got["h"]) and torch.equal(y, got["y"])  # without autograd
    return got


# rows of one to eight waves, 8 and 16 elements a lane, pieces that end early
SIZES = [(1, 1), (1, 2), (3, 7), (2, 8), (5, 64), (9, 65), (33, 100), (17, 511), (40, 512), (21, 520), (12, 771), (16, 1024), (7, 1025),
         (9, 1100), (6, 2048), (5, 2050), (4, 3000), (3, 4096), (3, 4100), (2, 8191), (2, 8192)]


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,d", SIZES)
def test_sizes(M, d, dtype, norm):
    verify(make(M, d, dtype, M + d, norm=norm))
    verify(make(M, d, dtype, M + d, parts=("scale",) if d % 2 else (), norm=norm, bias=norm == "layer"))


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("parts", [(), ("post",), ("gate",), ("scale",), ("post", "gate"), ("post", "scale"), ("gate", "scale"), ALL])
def test_parts(parts, norm):
    for dtype, wdtype in ((torch.bfloat16, None), (torch.float16, torch.float32), (torch.float32, None)):
        for alpha in (1.0, -0.5, 0.0):
            verify(make(20, 136, dtype, 3, parts, norm, alpha, wdtype))


def test_many_rows():
    """Every workgroup walks several rows, and the partial sums are many."""
    for d in (64, 1000):
        verify(make(6000, d, torch.bfloat16, 4))
        verify(make(6001, d, torch.float16, 5, parts=("gate",), norm="rms"))


@pytest.mark.parametrize("leaves", [("x",), ("r",), ("gate",), ("w",), ("b",), ("pw",), ("pb",), ("scale",), ("b", "scale")])
def test_only_some_gradients(leaves):
    got = verify(make(50, 72, torch.float16, 11), leaves)
    assert set(got) == {"h", "y"} | {"d" + k for k in leaves}


@pytest.mark.parametrize("parts", [(), ALL])
def test_only_one_result_is_used(parts):
    s = make(30, 96, torch.float32, 12, parts)
    want, err = exact({**s, "dy": None})
    got = run(s, outputs=("h",))
    for k in ("x", "r", "gate", "pw", "pb", "scale"):
        if s[k] is not None:
            check("d" + k, got["d" + k], want["d" + k], err["d" + k])
    assert got["dw"] is None and got["db"] is None
    want, err = exact({**s, "dh": None})
    got = run(s, outputs=("y",))
    for k in ROWS + VECTORS:
        if s[k] is not None:
            check("d" + k, got["d" + k], want["d" + k], err["d" + k])


def test_views_and_leading_dims():
    s = make(24, 40, torch.float16, 5)
    want, err = exact(s)
    t = {k: s[k].cuda() for k in ROWS + VECTORS}
    for name in ROWS:  # rows beside others, which are never used; columns first; rows from any element on
        wide = torch.full((24, 67), float("nan"), dtype=torch.float16, device="cuda")
        wide[:, 5:45] = t[name]
        for view in (wide[:, 5:45], t[name].t().contiguous().t()):
            h, y = call({**t, name: view}, s)
            check("h", h, want["h"], err["h"])
            check("y", y, want["y"], err["y"])
    u = {k: (v.view(2, 3, 4, 40) if k in ROWS else v).detach().requires_grad_(True) for k, v in t.items()}
    h, y = call(u, s)
    assert h.shape == y.shape == (2, 3, 4, 40)
    dh, dy = (s[k].cuda().t().contiguous().t().view(2, 3, 4, 40) for k in ("dh", "dy"))
    for k, v in zip(u, torch.autograd.grad((h, y), list(u.values()), (dh, dy))):
        check("d" + k, v.reshape(want["d" + k].shape), want["d" + k], err["d" + k])
    # one gate for all rows of a sequence: its gradient is their sum
    gate = s["gate"][:2].cuda().requires_grad_(True)
    rows = gate[:, None, :].expand(2, 12, 40)
    h, y = call({**{k: v.view(2, 12, 40) if k in ROWS else v for k, v in t.items()}, "gate": rows}, s)
    (dg,) = torch.autograd.grad((h, y), gate, (s["dh"].cuda().view(2, 12, 40), s["dy"].cuda().view(2, 12, 40)))
    want, err = exact({**s, "gate": s["gate"][:2, None].expand(2, 12, 40).reshape(24, 40)})
    u_ = UNIT[torch.float16]
    total = want["dgate"].view(2, 12, 40)
    tol = (u_ * total.abs() + err["dgate"].view(2, 12, 40)).sum(1) * 1.01 + 13 * u_ * total.abs().sum(1)
    assert ((dg.cpu().double() - total.sum(1)).abs() <= tol).all()


def test_one_tensor_in_several_places():
    s = make(20, 48, torch.float32, 6, ())
    x = s["x"].cuda().requires_grad_(True)
    t = {k: None if s[k] is None else s[k].cuda() for k in ROWS + VECTORS} | {"x": x, "r": x}
    h, y = call(t, s)
    (dx,) = torch.autograd.grad((h, y), x, (s["dh"].cuda(), s["dy"].cuda()))
    want, err = exact({**s, "r": s["x"]})
    check("dx", dx, want["dx"] + want["dr"], err["dx"] + err["dr"] + F32 * (want["dx"].abs() + want["dr"].abs()))


def test_no_rows():
    s = make(0, 24, torch.bfloat16, 1)
    got = run(s)
    for k in VECTORS:
        assert got["d" + k].shape == (24,) and not got["d" + k].any()
    assert got["h"].shape == got["dx"].shape == (0, 24)


def test_rows_that_are_not_finite_stay_alone():
    for M, d in ((12, 40), (12, 700), (12, 3000)):
        for norm in ("layer", "rms"):
            s = make(M, d, torch.bfloat16, 8, norm=norm)
            clean = run(s, ROWS)
            for k in ROWS:
                t = dict(s)
                t[k] = s[k].clone()
                t[k][3, d // 2], t[k][7, 0] = float("nan"), float("inf")
                got = run(t, ROWS)
                keep = [i for i in range(M) if i not in (3, 7)]
                for n in got:
                    assert torch.equal(got[n][keep], clean[n][keep]), (k, n)
                assert not torch.isfinite(got["y"][3]).any()


def test_large_mean():
    """Rows whose mean is 100 deviations away: the variance is that of centred values."""
    s = make(10, 300, torch.float32, 9, ("post",))
    s["x"] = s["x"] + 100
    s["r"] = s["r"] - 200
    verify(s)


def test_constant_rows():
    s = make(6, 80, torch.float32, 10, ("post",))
    s["x"][:] = 3.0
    s["r"][:] = 0.25
    got = run(s)
    assert all(torch.isfinite(v).all() for v in got.values())


@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_gradient_against_differences(norm):
    s = make(7, 20, torch.float32, 31, norm=norm, alpha=1.5)
    got = run(s)
    args = {k: s[k].double() for k in ROWS + VECTORS}

    def f(**a):
        t = {**s, **a}
        out, _ = exact(t)
        return (out["h"] * s["dh"].double()).sum() + (out["y"] * s["dy"].double()).sum()

    g = torch.Generator().manual_seed(2)
    for k in args:
        d = torch.randn(args[k].shape, generator=g, dtype=torch.float64)
        e = 1e-5
        up, dn = (f(**{n: t + sign * e * d if n == k else t for n, t in args.items()}) for sign in (1, -1))
        mine = got["d" + k].cpu().double() * d
        # float32 throughout (2^-24 times some hundreds) and the differences' own error of e^2
        assert abs(mine.sum() - (up - dn) / (2 * e)) <= 1e-4 * mine.abs().sum(), k


HOOKS = [(lambda t: t.cpu(), lambda t: t.cuda()), (lambda t: t, lambda t: t.contiguous().clone()),
         (lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone())]


@pytest.mark.parametrize("pack,unpack", HOOKS)
def test_saved_tensors_in_another_layout(pack, unpack):
    s = make(40, 72, torch.float16, 14)
    for fn in (None, _ResidualNormFn.apply):
        want = run(s, fn=fn)
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            got = run(s, fn=fn)
        assert all(torch.equal(got[k], want[k]) for k in want)


def test_both_paths_agree():
    for parts in ((), ALL):
        s = make(60, 200, torch.bfloat16, 21, parts)
        a, b = run(s), run(s, fn=_ResidualNormFn.apply)
        assert all(torch.equal(a[k], b[k]) for k in a)


def test_gradients_are_not_differentiable_again():
    s = make(20, 16, torch.float32, 3, ())
    t = {k: None if s[k] is None else s[k].cuda() for k in ROWS + VECTORS}
    x = t["x"].requires_grad_(True)
    for rows in (x, x.t().contiguous().t()):
        h, y = call({**t, "x": rows}, s)
        (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            dx.square().sum().backward()


def test_backward_twice_and_changed_operands():
    s = make(30, 40, torch.bfloat16, 13)
    t = {k: s[k].cuda().requires_grad_(True) for k in ROWS + VECTORS}
    h, y = call(t, s)
    leaves = list(t.values())
    first = torch.autograd.grad((h.sum() + y.sum()), leaves, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad((h.sum() + y.sum()), leaves)))
    h, y = call(t, s)
    with torch.no_grad():
        t["r"].add_(1)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), leaves)
    # h is the next block's residual: written over, it leaves these gradients alone
    h, y = call(t, s)
    want = torch.autograd.grad(y.sum(), leaves, retain_graph=True)
    h.detach().zero_()
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(y.sum(), leaves)))


def test_repeats_bit_for_bit_and_on_another_stream():
    s = make(3000, 200, torch.bfloat16, 8)
    a = run(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run(s)
    side.synchronize()
    assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("M,d", [(32, 768), (700, 300)])
def test_graph_replays(M, d):
    """Forward and backward in one graph, replayed with eager calls between."""
    s = make(M, d, torch.float16, 12)
    t = {k: s[k].cuda().requires_grad_(True) for k in ROWS + VECTORS}
    dh, dy = s["dh"].cuda(), s["dy"].cuda()

    def step():
        h, y = call(t, s)
        return [h.detach(), y.detach(), *torch.autograd.grad((h, y), list(t.values()), (dh, dy))]

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
            t["x"].copy_(make(M, d, torch.float16, 40 + seed)["x"])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals():
    x = torch.zeros(4, 16, device="cuda", dtype=torch.float16)
    w = torch.zeros(16, device="cuda", dtype=torch.float16)
    for bad in (dict(norm="batch"), dict(post_weight=w), dict(post_bias=w), dict(residual_scale=float("nan"))):
        with pytest.raises(ValueError):
            fm.residual_norm(x, x, w, w, **bad)
    for bad in (dict(residual=x[:3]), dict(weight=w[:8]), dict(gate=x[:, :8]), dict(scale=x), dict(gate=x[:, :1])):
        with pytest.raises(AssertionError):
            fm.residual_norm(**({"x": x, "residual": x, "weight": w} | bad))
    for bad in (dict(residual=x.float()), dict(weight=w.bfloat16()), dict(weight=w, scale=w.float()), dict(gate=x.bfloat16())):
        with pytest.raises(TypeError):
            fm.residual_norm(**({"x": x, "residual": x} | bad))
    with pytest.raises(TypeError):
        fm.residual_norm(x.double(), x.double())
    for bad in (dict(x=x.cpu()), dict(residual=x.cpu()), dict(weight=w.cpu()), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(RuntimeError):
            fm.residual_norm(**({"x": x, "residual": x} | bad))
    wide = torch.zeros(1, 8193, device="cuda")
    with pytest.raises(RuntimeError, match="MAX_D"):
        fm.residual_norm(wide, wide)


def test_views_read_with_their_sign():
    s = {k: v.cuda() if torch.is_tensor(v) else v for k, v in make(30, 24, torch.float16, 6).items()}
    got, want = [], []
    for out, f in ((got, torch._neg_view), (want, lambda t: -t)):
        t = {k: f(s[k]).detach().requires_grad_(True) for k in ROWS + VECTORS}
        h, y = call(t, s)
        out += [h, y, *torch.autograd.grad((h, y), list(t.values()), (f(s["dh"]), f(s["dy"])))]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tangents_refused():
    x = torch.randn(4, 16, device="cuda")
    w = torch.randn(16, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        t, u = torch.autograd.forward_ad.make_dual(x, x), torch.autograd.forward_ad.make_dual(w, w)
        for f in (lambda: fm.residual_norm(t, x), lambda: fm.residual_norm(x, t), lambda: fm.residual_norm(x, x, u),
                  lambda: fm.residual_norm(x, x, gate=t), lambda: fm.residual_norm(x, x, scale=u)):
            with pytest.raises(NotImplementedError):
                f()
        inside = fm.residual_norm(x, x, w)
    assert all(torch.equal(a, b) for a, b in zip(inside, fm.residual_norm(x, x, w)))
