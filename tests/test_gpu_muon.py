"""orthogonalize, muon_step and Muon against the iteration in 64 bits.

The kernels round fp16 operands (X's upper half, A and B = a I + b A + c A^2) and keep X as a pair of fp16
values, everything else in 32 bits. What that costs depends on the singular values; `emulated` is the same iteration
in 64 bits with those roundings, and the kernels may be twice as far from the formula as it is (their sums in
32 bits round some operands the other way) and 2^-16 of the norm more (2^-24 for each of up to 4096 / 16 terms that
one accumulator adds). The result's own rounding is u of each element.
"""

from __future__ import annotations

import copy
import math
import pickle

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_muon import COEFFICIENTS

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def iterate(u, rounded, steps=5, eps=1e-7, coefficients=COEFFICIENTS):
    """The formula in 64 bits, with or without the kernels' roundings."""
    a, b, c = coefficients

    def half(t, by):
        return (t * by).half().double() / by if rounded else t

    x = u.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / max(float(x.norm()), eps)
    for _ in range(steps):
        hi = half(x, 256.0)
        x = hi + half(x - hi, 256.0)  # (without the roundings hi is x)
        A = half(hi @ hi.t(), 1024.0)
        B = half(a * torch.eye(len(A)).to(A) + b * A + c * A @ A, 1024.0)
        x = B @ hi + a * (x - hi)
    return x.t() if tall else x


def tolerance(u, **kw):
    """(the result, how far off the norm of the kernels' may be)"""
    want = iterate(u, False, **kw)
    return want, 2 * float((iterate(u, True, **kw) - want).norm()) + 2.0 ** -16 * float(want.norm())


def check(got, u, **kw):
    want, tol = tolerance(u.cpu(), **kw)
    assert got.shape == u.shape and got.dtype == u.dtype
    off = float((got.cpu().double() - want).norm())
    tiny = 2.0 ** -25 * math.sqrt(want.numel()) if got.dtype == torch.float16 else 0.0
    tol += UNIT[got.dtype] * float(want.norm()) + tiny
    assert off <= tol, f"{tuple(u.shape)}: off by {off}, tolerance {tol}, norm {float(want.norm())}"


def matrix(rows, cols, kind, seed):
    g = torch.Generator().manual_seed(seed)
    r = min(rows, cols)
    if kind == "gauss":
        return torch.randn(rows, cols, generator=g)
    if kind == "rank one":
        return torch.randn(rows, 1, generator=g) @ torch.randn(1, cols, generator=g)
    fall = torch.arange(1, r + 1).float() ** -1.0
    return (torch.randn(rows, r, generator=g) * fall) @ torch.randn(r, cols, generator=g)


SHAPES = [(1, 1), (1, 9), (9, 1), (2, 2), (3, 5), (33, 17), (64, 64), (65, 63), (63, 65), (128, 300), (300, 128), (257, 511),
          (512, 130), (1000, 24), (24, 1000), (500, 500)]


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_shapes(rows, cols, dtype):
    u = matrix(rows, cols, "falling" if rows % 2 else "gauss", rows + cols).to(dtype).cuda()
    before = u.clone()
    check(fm.orthogonalize(u), u)
    assert torch.equal(u, before)


@pytest.mark.parametrize("rows,cols", [(128, 768), (768, 128), (300, 300)])
@pytest.mark.parametrize("kind", ["gauss", "rank one", "falling"])
def test_spectra(kind, rows, cols):
    u = matrix(rows, cols, kind, 3).cuda()
    check(fm.orthogonalize(u), u)


@pytest.mark.parametrize("rows,cols", [(1024, 4096), (4096, 1024), (2000, 1500)])
@pytest.mark.parametrize("count", [1, 9])
def test_large_tiles(rows, cols, count):
    """Each tile size, in both directions: against the formula in 64 bits on the GPU (2e-3 of the norm, of a Gaussian
    matrix's 1.3e-3 to 1.5e-3 by emulation, and the rounding to bfloat16)."""
    g = torch.Generator(device="cuda").manual_seed(1)
    us = [torch.randn(rows, cols, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(count)]
    for u, got in zip(us, fm.orthogonalize(us)):
        want = iterate(u, False)
        assert (got.double() - want).norm() <= (2e-3 + 2.0 ** -8) * want.norm()


def test_tiles_of_many_shapes_one_after_the_other():
    """Workgroups that go from tile to tile through matrices of other sizes: sides that end inside a tile, an odd count of
    stages, tall ones, one too small for the tile; one of them three times."""
    g = torch.Generator(device="cuda").manual_seed(2)
    sizes = [(1024, 4096)] * 3 + [(320, 20000), (5000, 450), (40, 3000), (700, 9000), (1000, 130)]
    us = [torch.randn(*s, generator=g, device="cuda") for s in sizes]
    us += [us[4]] * 2
    results = fm.orthogonalize(us)
    for u, got in zip(us, results):
        want, tol = tolerance(u)
        assert (got.double() - want).norm() <= tol + UNIT[got.dtype] * want.norm(), u.shape
    assert torch.equal(results[4], results[-1]) and torch.equal(results[4], results[-2])


@pytest.mark.parametrize("rows,cols", [(64, 1000), (100, 600), (190, 300), (256, 1024), (1000, 200), (250, 70)])
def test_small_matrices_alone_and_among_many(rows, cols):
    """Alone, B has no launch of its own; among forty it has. The same bits."""
    u = matrix(rows, cols, "falling", 8).cuda()
    alone = fm.orthogonalize(u)
    check(alone, u)
    assert all(torch.equal(o, alone) for o in fm.orthogonalize([u] * 40))


def test_scales():
    """The result does not depend on the update's size, until its norm is below eps."""
    u = matrix(60, 90, "gauss", 5)
    for by in (1e-25, 1e-6, 1.0, 1e6, 1e30):
        check(fm.orthogonalize((u * by).cuda(), eps=1e-30), u)
    check(fm.orthogonalize((u * 1e-12).cuda()), u * 1e-12)  # norm below eps
    check(fm.orthogonalize(u.cuda(), eps=1e3), u, eps=1e3)
    assert not fm.orthogonalize(torch.zeros(8, 8, device="cuda"), eps=1e-60).any()


def test_steps_and_coefficients():
    u = matrix(70, 200, "falling", 6)
    for steps in (1, 2, 3, 6):
        check(fm.orthogonalize(u.cuda(), steps=steps), u, steps=steps)
    other = (1.875, -1.25, 0.375)  # converges to the polar factor
    check(fm.orthogonalize(u.cuda(), steps=12, coefficients=other), u, steps=12, coefficients=other)


def test_many_matrices_of_all_shapes():
    """More than a launch's table holds, empty ones and ones of other types among them; each as if alone."""
    g = torch.Generator().manual_seed(7)
    us = [torch.randn(int(r), int(c), generator=g).cuda()
          for r, c in torch.randint(0, 150, (95, 2), generator=g).tolist() + [[700, 900]]]
    us[3], us[50] = us[3].bfloat16(), us[50].half()
    got = fm.orthogonalize(us)
    for u, o in zip(us, got):
        assert o.shape == u.shape and o.dtype == u.dtype
        if u.numel():
            check(o, u)
            assert torch.equal(o, fm.orthogonalize(u)) or u.numel() > 100 * 100  # (tiles may differ for large ones)
    assert fm.orthogonalize([]) == []


def test_zeros_and_values_that_are_not_finite():
    us = [torch.randn(40, 70, device="cuda") for _ in range(4)]
    us[1].zero_()
    us[2][3, 4] = float("nan")
    us[3][0, 0] = float("inf")
    got = fm.orthogonalize(us)
    assert not got[1].any() and torch.isnan(got[2]).all() and not torch.isfinite(got[3]).all()
    check(got[0], us[0])


def test_views():
    u = torch.randn(50, 80, device="cuda")
    want = fm.orthogonalize(u)
    assert torch.equal(fm.orthogonalize(u.t().contiguous().t()), want)
    assert torch.equal(fm.orthogonalize(torch._neg_view(u)), fm.orthogonalize(-u))
    check(fm.orthogonalize(torch._neg_view(u)), -u)
    odd = torch.empty(50 * 80 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(50, 80).copy_(u)
    assert torch.equal(fm.orthogonalize(odd), fm.orthogonalize(u.bfloat16()))


# ---- the step ----

def step_inputs(shapes, dtype, seed, grad_dtype=None):
    g = torch.Generator().manual_seed(seed)
    p = [(0.03 * torch.randn(s, generator=g)).to(dtype) for s in shapes]
    gr = [(1e-3 * torch.randn(s, generator=g)).to(grad_dtype or dtype) for s in shapes]
    m = [1e-3 * torch.randn(s, generator=g) for s in shapes]
    return p, gr, m


def step_check(p0, g, m0, p1, m1, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.1, adjust="original", scale=1.0):
    g = g.double() * scale
    m = momentum * m0.double() + (1 - momentum) * g
    # two products and a sum, and the constants: 2^-22 of the terms
    assert ((m1.cpu().double() - m).abs() <= 2.0 ** -22 * (m0.double().abs() + g.abs())).all()
    u = (1 - momentum) * g + momentum * m if nesterov else m
    o, tol = tolerance(u)
    r, c = u.shape
    rate = lr * (math.sqrt(max(1.0, r / c)) if adjust == "original" else 0.2 * math.sqrt(max(r, c)))
    p = p0.double() * (1 - lr * weight_decay) - rate * o
    off = float((p1.cpu().double() - p).norm())
    assert off <= rate * tol + (UNIT[p0.dtype] + 3 * 2.0 ** -24) * float(p.norm()) + 2.0 ** -22 * rate * float(o.norm())


SETTINGS = [dict(), dict(lr=0.02, momentum=0.9, nesterov=False, weight_decay=0.0), dict(lr=0.05, adjust="match_rms_adamw"),
            dict(lr=0.0), dict(momentum=0.0)]


@pytest.mark.parametrize("dtype,grad_dtype", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, None),
                                              (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("kw", SETTINGS)
def test_step(kw, dtype, grad_dtype):
    shapes = [(96, 40), (40, 96), (128, 128), (7, 300), (130, 66)]
    p, g, m = step_inputs(shapes, dtype, 11, grad_dtype)
    P, G, M = ([t.cuda() for t in x] for x in (p, g, m))
    fm.muon_step(P, G, M, **kw)
    for i in range(len(shapes)):
        step_check(p[i], g[i], m[i], P[i], M[i], **kw)
        assert torch.equal(G[i].cpu(), g[i])


def test_step_scale_and_copies():
    shapes = [(70, 33), (33, 70)]
    p, g, m = step_inputs(shapes, torch.float32, 12, torch.bfloat16)
    P, G, M = ([t.cuda() for t in x] for x in (p, g, m))
    C = [torch.empty(70, 33, device="cuda", dtype=torch.bfloat16), None]
    fm.muon_step(P, G, M, lr=0.02, grad_scale=torch.full((), 0.25, device="cuda"), copies=C)
    for i in range(2):
        step_check(p[i], g[i], m[i], P[i], M[i], lr=0.02, scale=0.25)
    assert torch.equal(C[0], P[0].bfloat16())


def test_step_at_any_address():
    """Parameters, gradients and momenta that begin at any element, rows of odd widths."""
    for r, c in ((37, 53), (53, 37)):
        p, g, m = step_inputs([(r, c)], torch.bfloat16, 13)

        def odd(t):
            return torch.full((r * c + 2,), 7.0, device="cuda", dtype=t.dtype)

        stores = [odd(t) for t in (p[0], g[0], m[0])]
        P, G, M = (s[1:-1].view(r, c).copy_(t) for s, t in zip(stores, (p[0], g[0], m[0])))
        fm.muon_step([P], [G], [M])
        step_check(p[0], g[0], m[0], P, M)
        assert all(s[0] == 7 and s[-1] == 7 for s in stores)


def test_repeats_bit_for_bit_and_on_another_stream():
    us = [torch.randn(r, c, device="cuda") for r, c in ((300, 500), (500, 300), (128, 128))]
    a = fm.orthogonalize(us)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = fm.orthogonalize(us)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_graph_replays():
    shapes = [(200, 70), (70, 200), (64, 64)]
    p, g, m = step_inputs(shapes, torch.float32, 14)
    P, G, M = ([t.cuda() for t in x] for x in (p, g, m))
    fm.muon_step(P, G, M, lr=0.01)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fm.muon_step(P, G, M, lr=0.01)
    eager = [[t.clone() for t in x] for x in (P, G, M)]
    for seed in range(3):
        for x, y, t in zip(G, eager[1], step_inputs(shapes, torch.float32, 20 + seed)[1]):
            x.copy_(t)
            y.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        fm.muon_step(*eager, lr=0.01)
        assert all(torch.equal(x, y) for a, b in zip((P, M), (eager[0], eager[2])) for x, y in zip(a, b))


def test_versions_and_no_gradients():
    p = torch.randn(8, 16, device="cuda", requires_grad=True)
    g, m = torch.randn(8, 16, device="cuda"), torch.zeros(8, 16, device="cuda")
    y = (p * p).sum()
    fm.muon_step([p], [g], [m])
    with pytest.raises(RuntimeError):  # p was changed after y had saved it
        y.backward()
    assert not fm.orthogonalize(p).requires_grad


def train(opt, params, grads, steps):
    for k in range(steps):
        for p, g in zip(params, grads[k]):
            p.grad = g
        opt.step()


def test_optimizer():
    shapes = [(40, 24), (24, 40), (30, 30)]
    grads = [[t.cuda() for t in step_inputs(shapes, torch.float32, 30 + k)[1]] for k in range(4)]

    def fresh():
        return [torch.nn.Parameter(t.cuda()) for t in step_inputs(shapes, torch.float32, 29)[0]]

    params = fresh()
    opt = fm.Muon([{"params": params[:1], "lr": 0.03}, {"params": params[1:]}], lr=0.01, weight_decay=0.05)
    train(opt, params, grads, 4)
    P = [p.detach().clone() for p in fresh()]
    M = [torch.zeros_like(p) for p in P]
    for k in range(4):
        fm.muon_step(P[:1], grads[k][:1], M[:1], lr=0.03, weight_decay=0.05)
        fm.muon_step(P[1:], grads[k][1:], M[1:], lr=0.01, weight_decay=0.05)
    assert all(torch.equal(a.detach(), b) for a, b in zip(params, P))

    # a loaded state, a deep copy and a pickle go on as the optimizer itself
    second = fresh()
    half = fm.Muon([{"params": second[:1], "lr": 0.03}, {"params": second[1:]}], lr=0.01, weight_decay=0.05)
    train(half, second, grads, 2)
    third = [torch.nn.Parameter(p.detach().clone()) for p in second]
    loaded = fm.Muon([{"params": third[:1]}, {"params": third[1:]}])
    loaded.load_state_dict(half.state_dict())
    fourth = copy.deepcopy(half)
    fifth = pickle.loads(pickle.dumps(half))
    for o in (loaded, fourth, fifth):
        mine = [p for g in o.param_groups for p in g["params"]]
        train(o, mine, grads[2:], 2)
        assert all(torch.equal(a.detach(), b) for a, b in zip(mine, P))


def test_optimizer_of_16_bits_keeps_float32_momenta():
    p = torch.nn.Parameter(torch.randn(16, 32, device="cuda", dtype=torch.bfloat16))
    opt = fm.Muon([p])
    train(opt, [p], [[torch.randn_like(p)]], 1)
    other = fm.Muon([torch.nn.Parameter(p.detach().clone())])
    other.load_state_dict(opt.state_dict())
    m = other.state[other.param_groups[0]["params"][0]]["momentum_buffer"]
    assert m.dtype == torch.float32 and torch.equal(m, opt.state[p]["momentum_buffer"])
    c = torch.empty(4, 4, device="cuda", dtype=torch.bfloat16)
    q = torch.nn.Parameter(torch.randn(4, 4, device="cuda"))
    with_copy = fm.Muon([q, p], copies=[c, None])
    train(with_copy, [q, p], [[torch.randn_like(q), torch.randn_like(p)]], 1)
    assert torch.equal(c, q.detach().bfloat16())
    again = copy.deepcopy(with_copy)
    assert list(again._copies.values())[0].shape == c.shape


def test_state_of_torch_continues():
    """torch.optim.Muon iterates in bfloat16: one step of it from the same state is within 5 % of the update."""
    p = torch.nn.Parameter(torch.randn(48, 96, device="cuda") * 0.03)
    theirs = torch.optim.Muon([p], lr=0.02, weight_decay=0.0)
    for k in range(2):
        p.grad = torch.randn(48, 96, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda")
        theirs.step()
    q = torch.nn.Parameter(p.detach().clone())
    mine = fm.Muon([q])
    mine.load_state_dict(theirs.state_dict())
    assert mine.param_groups[0]["steps"] == 5 and mine.param_groups[0]["adjust"] == "original"
    before = p.detach().clone()
    p.grad = torch.randn(48, 96, device="cuda")
    q.grad = p.grad.clone()
    theirs.step()
    mine.step()
    assert (p - q).norm() <= 0.05 * (p - before).norm()


def test_refusals():
    p, m = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    g = torch.ones(4, 8, device="cuda")
    ok = dict(params=[p], grads=[g], momenta=[m])
    for bad in (dict(adjust="other"), dict(grads=[]), dict(params=[p.t().contiguous().t()]), dict(coefficients=(1.0, 2.0)),
                dict(momenta=[p]), dict(momenta=[g]), dict(grads=[p]), dict(params=[p, p], grads=[g, g], momenta=[m, m.clone()])):
        with pytest.raises(ValueError):
            fm.muon_step(**(ok | bad))
    for bad in (dict(grads=[g[:3]]), dict(momenta=[m.view(8, 4)]), dict(params=[p[0]], grads=[g[0]], momenta=[m[0]]),
                dict(grad_scale=torch.ones(2, device="cuda"))):
        with pytest.raises(AssertionError):
            fm.muon_step(**(ok | bad))
    for bad in (dict(momenta=[m.half()]), dict(params=[p.double()]), dict(params=[p.half()], grads=[g.bfloat16()]),
                dict(copies=[torch.zeros_like(p)]), dict(grad_scale=torch.ones((), device="cuda", dtype=torch.float64)),
                dict(copies=[torch.zeros(4, 8, device="cuda", dtype=torch.half)], grads=[g.bfloat16()])):
        with pytest.raises(TypeError):
            fm.muon_step(**(ok | bad))
    for bad in (dict(momentum=1.0), dict(lr=-1.0), dict(steps=0), dict(eps=0.0), dict(coefficients=(1.0, float("nan"), 0.0)),
                dict(coefficients=(21.0, 0.0, 0.0)),
                dict(grads=[g.cpu()]), dict(weight_decay=float("nan"))):
        with pytest.raises(RuntimeError):
            fm.muon_step(**(ok | bad))
    assert not p.any() and not m.any()
    flat = torch.zeros(96, device="cuda")
    with pytest.raises(ValueError, match="share"):  # the momentum's last row is the parameter's first
        fm.muon_step([flat[24:56].view(4, 8)], [g], [flat[:32].view(4, 8)])
    fm.muon_step([flat[:32].view(4, 8)], [flat[64:].view(4, 8)], [flat[32:64].view(4, 8)])  # side by side
    # one matrix past the limits among others of another type: none is moved
    q, big = torch.ones(4, 8, device="cuda", dtype=torch.half), torch.zeros((1 << 20) + 1, 1, device="cuda")
    with pytest.raises(ValueError, match="sides"):
        fm.muon_step([q, big], [torch.ones_like(q), big + 1], [m.clone(), big + 2])
    assert (q == 1).all()
    with pytest.raises(AssertionError):
        fm.orthogonalize(p[0])
    with pytest.raises(TypeError):
        fm.orthogonalize(p.double())
    with pytest.raises(ValueError):
        fm.Muon([torch.nn.Parameter(torch.zeros(4, device="cuda"))])
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(g, g)
        with pytest.raises(NotImplementedError):
            fm.orthogonalize(t)
        with pytest.raises(NotImplementedError):
            fm.muon_step([p], [t], [m])
