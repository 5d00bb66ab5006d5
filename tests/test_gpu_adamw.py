"""adamw_step, AdamW and the 8-bit moments against plain implementations.

float32 moments: two products and a sum, each rounded, so m is off by at most
4 * 2^-24 of its terms' magnitudes and v likewise; the step multiplies a root, a
reciprocal (one ulp) and two products more, 16 * 2^-24 of it; the parameter adds
its own rounding. 8-bit moments follow a formula whose every operation is rounded
to float32, so codes and scales equal the same formula's in torch exactly; its
root is the GPU's, which torch takes there too (the CPU's differs in the last bit
now and then).
"""

from __future__ import annotations

import copy
import math

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_optim import BLOCK

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: F32}
HP = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def make(n, dtype, gdtype, seed):
    g = torch.Generator().manual_seed(seed)
    p = (0.1 * torch.randn(n, generator=g)).to(dtype)
    gr = (0.01 * torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g))).to(gdtype)
    m = 0.005 * torch.randn(n, generator=g)
    v = (0.01 * torch.randn(n, generator=g)) ** 2
    return p, gr, m, v


def exact(p, g, m, v, step, scale=1.0, lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1):
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * scale
    m1 = betas[0] * m + (1 - betas[0]) * g
    v1 = betas[1] * v + (1 - betas[1]) * g * g
    upd = lr * (m1 / (1 - betas[0] ** step)) / (torch.sqrt(v1 / (1 - betas[1] ** step)) + eps)
    me = 4 * F32 * ((betas[0] * m).abs() + ((1 - betas[0]) * g).abs())
    ve = 4 * F32 * v1
    pe = 16 * F32 * upd.abs() + 4 * F32 * p.abs() + upd.abs() * me / m1.abs().clamp(min=1e-30)
    return p * (1 - lr * weight_decay) - upd, m1, v1, pe, me, ve


def within(got, want, err):
    got = got.detach().cpu()
    tol = UNIT[got.dtype] * want.abs() + err + (2.0 ** -25 if got.dtype == torch.float16 else 1e-38)
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"off by {off.max().item()}, {(off / tol).max().item()} of the tolerance"


def encode(x, signed):
    """Codes and scales of the blocks of x, in torch: every operation rounded to float32."""
    n, top = x.numel(), 127 if signed else 255
    b = torch.nn.functional.pad(x, (0, -n % BLOCK)).view(-1, BLOCK)
    big = b.abs().amax(1, keepdim=True)
    whole = torch.full_like(big, float(top * top))
    tiny = big < 2.0 ** -110
    y = b.abs() * torch.where(tiny, torch.zeros_like(big), whole / torch.where(tiny, torch.ones_like(big), big))
    mid = (torch.arange(1, top + 1, device=x.device) - 0.5).square()  # code c from (c - 1/2)^2 on
    c = torch.bucketize(y, mid, right=True)
    c = torch.where((b > 0) & ~tiny & (not signed), c.clamp(min=1), c)
    c = torch.where(b < 0, -c, c).to(torch.int8 if signed else torch.uint8)
    return c.view(-1)[:n], (torch.where(tiny, torch.zeros_like(big), big) / whole).view(-1)


def decode(c, q):
    f = c.float()
    return f * f.abs() * q.repeat_interleave(BLOCK)[: c.numel()]


def plain8(p, g, m8, v8, step, scale, hp):
    """One step in torch, in float32, each operation by itself."""
    b1, b2 = hp["betas"]
    g = g.float() * scale
    root = decode(*v8)
    m = decode(*m8) * b1 + g * (1 - b1)
    v = (root * root) * b2 + (g * g) * (1 - b2)
    root = torch.sqrt(v.cuda()).cpu()
    upd = m / (root * (1 / math.sqrt(1 - b2 ** step)) + hp["eps"]) * (hp["lr"] / (1 - b1 ** step))
    p = p.float() * (1 - hp["lr"] * hp["weight_decay"]) - upd
    return p, encode(m, True), encode(root, False), upd.abs()


@pytest.mark.parametrize("n", [1, 7, 255, 256, 257, 2048, 2049, 70001])
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                   (torch.float16, torch.float16), (torch.bfloat16, torch.float32),
                                   (torch.float16, torch.float32), (torch.float32, torch.bfloat16),
                                   (torch.float32, torch.float16)])
def test_float32_moments(n, types):
    p, g, m, v = make(n, *types, n)
    want = exact(p, g, m, v, 3, **HP)
    P, G, Mo, V = (t.cuda() for t in (p, g, m, v))
    fm.adamw_step([P], [G], [Mo], [V], 3, **HP)
    for got, w, e in zip((P, Mo, V), want, want[3:]):
        within(got, w, e)


@pytest.mark.parametrize("ctype", [torch.float16, torch.bfloat16])
def test_copies_and_grad_scale(ctype):
    p, g, m, v = make(5000, torch.float32, torch.float32, 4)
    want = exact(p, g, m, v, 7, scale=0.25, **HP)
    P, G, Mo, V = (t.cuda() for t in (p, g, m, v))
    C = torch.full((5000,), 9.0, dtype=ctype, device="cuda")
    fm.adamw_step([P], [G], [Mo], [V], 7, grad_scale=torch.tensor(0.25, device="cuda"), copies=[C], **HP)
    within(P, want[0], want[3])
    assert torch.equal(C, P.to(ctype))


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_in_one_call(bits):
    """More than one launch holds; sizes of zero, one, off the blocks; mixed types; unaligned views."""
    g = torch.Generator().manual_seed(5)
    sizes = [0, 1, 3, 255, 256, 257, 4096] + torch.randint(1, 6000, (130,), generator=g).tolist()
    dtypes = [torch.float32, torch.bfloat16, torch.float16]
    lists, want = ([], [], [], []), []
    for i, n in enumerate(sizes):
        p, gr, m, v = make(n, dtypes[i % 3], torch.float32 if i % 5 == 0 else dtypes[i % 3], i)
        if bits == 8:
            ms, vs = encode(m, True), encode(v.sqrt(), False)
            want.append((p, gr, ms, vs))
            m, v = tuple(t.cuda() for t in ms), tuple(t.cuda() for t in vs)
        else:
            want.append(exact(p, gr, m, v, 2, **HP))
            m, v = m.cuda(), v.cuda()
        buf = torch.zeros(n + 3, dtype=p.dtype, device="cuda")
        view = buf[i % 4: i % 4 + n]
        view.copy_(p)
        for x, t in zip(lists, (view, gr.cuda(), m, v)):
            x.append(t)
    fm.adamw_step(*lists, 2, **HP)
    for (P, _, Mo, V), w in zip(zip(*lists), want):
        if bits == 32:
            for got, a, e in zip((P, Mo, V), w, w[3:]):
                within(got, a, e)
        elif P.numel():
            pe, ms, vs, upd = plain8(w[0], w[1], w[2], w[3], 2, 1.0, HP)
            assert all(torch.equal(a.cpu(), b) for a, b in zip((*Mo, *V), (*ms, *vs)))
            # the step by a reciprocal, 2^-22 of it; p rounded to its type
            within(P, pe.double(), 2.0 ** -22 * upd + 2 * F32 * pe.abs())


@pytest.mark.parametrize("n", [1, 31, 256, 300, 5003])
def test_8bit_moments_equal_the_formula(n):
    p, g, m, v = make(n, torch.float32, torch.float32, n + 1)
    m8, v8 = encode(m, True), encode(v.sqrt(), False)
    P, G = p.cuda(), g.cuda()
    M8, V8 = fm.AdamW8bitState(*(t.cuda() for t in m8)), fm.AdamW8bitState(*(t.cuda() for t in v8))
    tol = torch.zeros(n)
    for step in (1, 2, 3):
        p, m8, v8, upd = plain8(p, g, m8, v8, step, 0.5, HP)
        fm.adamw_step([P], [G], [M8], [V8], step, grad_scale=torch.full((1,), 0.5, device="cuda"), **HP)
        assert all(torch.equal(a.cpu(), b) for a, b in zip((*M8, *V8), (*m8, *v8)))
        tol += 2.0 ** -22 * upd + 2 * F32 * p.abs()  # the step by a reciprocal, and p's own rounding
        assert ((P.cpu() - p).abs() <= tol).all()
    assert torch.equal(fm.dequantize_adamw(M8).cpu(), decode(*m8))
    assert torch.equal(fm.dequantize_adamw(V8).cpu(), decode(*v8).square())


def test_8bit_moments_are_near_the_moments():
    """Half a step of the grid: (2 sqrt(y) + 1) / 2 of y = |m| / q at the nearest code."""
    p, g, m, v = make(40000, torch.float32, torch.float32, 77)
    m8, v8 = (tuple(torch.zeros_like(t).cuda() for t in s) for s in (encode(m, True), encode(v.sqrt(), False)))
    P = p.cuda()
    fm.adamw_step([P], [g.cuda()], [m8], [v8], 1, **HP)
    for got, x, s in ((fm.dequantize_adamw(m8).cpu(), 0.1 * g, m8), (fm.dequantize_adamw(v8).cpu().sqrt(), (0.01 * g * g).sqrt(), v8)):
        q = s[1].cpu().repeat_interleave(BLOCK)[: x.numel()]
        y = x.abs() / q
        if s is v8:  # a root that is not zero keeps code 1
            assert ((got - x).abs() <= q * torch.clamp(torch.sqrt(y) + 0.51, min=1.0) * 1.001).all()
            assert (got[x > 0] > 0).all()
        else:
            assert ((got - x).abs() <= q * (torch.sqrt(y) + 0.51) * 1.001).all()


def test_blocks_of_zeros_and_not_finite():
    n = 3 * BLOCK + 5
    p, g = torch.ones(n), torch.zeros(n)
    g[BLOCK + 3], g[2 * BLOCK] = float("inf"), float("nan")
    P, G = p.cuda(), g.cuda()
    m, v = fm.adamw_state(P, 8)
    fm.adamw_step([P], [G], [m], [v], 1, lr=0.1, weight_decay=0.0)
    md, vd = fm.dequantize_adamw(m).cpu(), fm.dequantize_adamw(v).cpu()
    for x in (md, vd):  # only the blocks of those values are lost
        assert not x[:BLOCK].any() and not x[3 * BLOCK:].any()
        assert not torch.isfinite(x[BLOCK:2 * BLOCK]).all() and not torch.isfinite(x[2 * BLOCK:3 * BLOCK]).all()
    got = P.cpu()
    finite = torch.isfinite(g)
    assert (got[finite] == 1).all() and torch.isnan(got[2 * BLOCK])
    # the smallest moments: held as zeros, never a division by zero
    P, G = torch.ones(300).cuda(), torch.full((300,), 1e-36).cuda()
    m, v = fm.adamw_state(P, 8)
    fm.adamw_step([P], [G], [m], [v], 1)
    assert torch.isfinite(P).all() and torch.isfinite(fm.dequantize_adamw(m)).all()


def test_optimizer_matches_the_steps_and_resumes():
    g = torch.Generator().manual_seed(6)
    shapes = [(33, 7), (300,), (1,), (64, 64)]
    init = [torch.randn(s, generator=g) for s in shapes]
    grads = [[torch.randn(s, generator=g) * 0.1 for s in shapes] for _ in range(4)]
    for bits in (32, 8):
        def fresh():
            ps = [torch.nn.Parameter(t.cuda().bfloat16() if i == 1 else t.cuda()) for i, t in enumerate(init)]
            return ps, fm.AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 5e-3}], state_bits=bits, **HP)

        def steps(ps, opt, which):
            for k in which:
                for i, p in enumerate(ps):  # the last parameter misses the second step
                    p.grad = None if (i == 3 and k == 1) else grads[k][i].cuda().to(p.dtype)
                opt.step()

        a, oa = fresh()
        steps(a, oa, range(4))
        b, ob = fresh()
        steps(b, ob, range(2))
        c, oc = fresh()
        oc.load_state_dict(copy.deepcopy(ob.state_dict()))
        for p, q in zip(c, b):
            p.data.copy_(q.data)
        steps(c, oc, range(2, 4))
        assert all(torch.equal(p, q) for p, q in zip(a, c))
        assert [oa.state[p]["step"] for p in a] == [4, 4, 4, 3]
        assert oc.state[c[1]]["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.int8)
        if bits == 32:
            p, m, v = init[0].double().flatten(), torch.zeros(231), torch.zeros(231)
            for k in range(4):
                p, m, v = exact(p, grads[k][0].flatten(), m, v, k + 1, **HP)[:3]
            assert (a[0].detach().cpu().double().flatten() - p).abs().max() <= 4 * 20 * F32 * p.abs().max()


def test_optimizer_copies_versions_and_zero_sizes():
    p = torch.nn.Parameter(torch.randn(100, device="cuda"))
    e = torch.nn.Parameter(torch.empty(0, device="cuda"))
    c = torch.zeros(100, dtype=torch.bfloat16, device="cuda")
    opt = fm.AdamW([p, e], copies=[c, None])
    p.grad, e.grad = torch.randn(100, device="cuda"), torch.empty(0, device="cuda")
    before = p._version
    opt.step(grad_scale=torch.ones((), device="cuda"))
    assert p._version > before and torch.equal(c, p.detach().bfloat16())


def test_graph_replays():
    p, g, m, v = (t.cuda() for t in make(3000, torch.float32, torch.float32, 9))
    G = torch.cuda.CUDAGraph()
    p0, m0, v0 = p.clone(), m.clone(), v.clone()
    fm.adamw_step([p0], [g], [m0], [v0], 5, **HP)
    torch.cuda.synchronize()
    with torch.cuda.graph(G):
        fm.adamw_step([p], [g], [m], [v], 5, **HP)
    for _ in range(3):
        G.replay()
        torch.cuda.synchronize()
        assert torch.equal(p, p0) and torch.equal(m, m0) and torch.equal(v, v0)
        fm.adamw_step([p0], [g], [m0], [v0], 5, **HP)
        torch.cuda.synchronize()


def test_refusals():
    p, g, m, v = (t.cuda() for t in make(300, torch.float32, torch.float32, 1))
    m8, v8 = fm.adamw_state(p, 8)
    with pytest.raises(ValueError):
        fm.adamw_step([p], [g], [m], [v, v], 1)
    with pytest.raises(ValueError):
        fm.adamw_step([p, p], [g, g], [m, m8], [v, v8], 1)
    with pytest.raises(ValueError):
        fm.adamw_step([p], [g], [m[:299]], [v], 1)
    with pytest.raises(ValueError):
        fm.adamw_step([p], [g], [fm.AdamW8bitState(m8[0], m8[1][:1])], [v8], 1)
    with pytest.raises(ValueError):
        fm.adamw_step([p.view(20, 15).t()], [g.view(20, 15).t()], [m], [v], 1)
    with pytest.raises(AssertionError):
        fm.adamw_step([p], [g[:200]], [m], [v], 1)
    with pytest.raises(TypeError):
        fm.adamw_step([p.double()], [g], [m], [v], 1)
    with pytest.raises(TypeError):
        fm.adamw_step([p.half()], [g.bfloat16()], [m], [v], 1)
    with pytest.raises(TypeError):
        fm.adamw_step([p], [g], [m.half()], [v], 1)
    with pytest.raises(TypeError):
        fm.adamw_step([p], [g], [v8], [m8], 1)
    with pytest.raises(TypeError):
        fm.adamw_step([p.half()], [g], [m], [v], 1, copies=[p.half()])
    with pytest.raises(TypeError):
        fm.adamw_step([p], [g], [m], [v], 1, grad_scale=torch.ones((), device="cuda").double())
    with pytest.raises(RuntimeError):
        fm.adamw_step([p.cpu()], [g], [m], [v], 1)
    with pytest.raises(RuntimeError, match="step"):
        fm.adamw_step([p], [g], [m], [v], 0)
    with pytest.raises(RuntimeError, match="betas"):
        fm.adamw_step([p], [g], [m], [v], 1, betas=(1.0, 0.9))
    with pytest.raises(ValueError):
        fm.AdamW([torch.nn.Parameter(p)], state_bits=16)
    with pytest.raises(ValueError):
        fm.AdamW([torch.nn.Parameter(p)], lr=-1.0)
    with pytest.raises(ValueError):
        fm.AdamW([torch.nn.Parameter(p)], copies=[None, None])
    with pytest.raises(TypeError):
        fm.dequantize_adamw((p, m8[1]))


def test_gradients_read_with_their_sign():
    p = [torch.ones(300, device="cuda"), torch.ones(300, device="cuda")]
    g = torch.linspace(-1, 1, 300, device="cuda")
    for q, h in zip(p, (torch._neg_view(g), -g)):
        m, v = fm.adamw_state(q)
        fm.adamw_step([q], [h], [m], [v], 1)
    assert torch.equal(*p)
    with pytest.raises(ValueError):
        fm.adamw_step([torch._neg_view(p[0])], [g], [torch.zeros_like(g)], [torch.zeros_like(g)], 1)


def test_optimizer_continues_torchs_state():
    g = torch.Generator().manual_seed(9)
    init, grads = torch.randn(50, 7, generator=g), [torch.randn(50, 7, generator=g) for _ in range(3)]
    a, b = (torch.nn.Parameter(init.cuda()) for _ in range(2))
    theirs = torch.optim.AdamW([a], **HP)
    for k in range(2):
        a.grad = grads[k].cuda()
        theirs.step()
    mine = fm.AdamW([b])
    mine.load_state_dict(copy.deepcopy(theirs.state_dict()))
    b.data.copy_(a.data)
    want = exact(a.detach().cpu().double().flatten(), grads[2].flatten(), theirs.state[a]["exp_avg"].cpu().flatten(),
                 theirs.state[a]["exp_avg_sq"].cpu().flatten(), 3, **HP)[0]
    b.grad = grads[2].cuda()
    mine.step()
    assert type(mine.state[b]["step"]) is int and mine.state[b]["step"] == 3
    assert (b.detach().cpu().double().flatten() - want).abs().max() <= 20 * F32 * want.abs().max()
    with pytest.raises(ValueError):
        mine.load_state_dict(torch.optim.AdamW([a], amsgrad=True).state_dict())
