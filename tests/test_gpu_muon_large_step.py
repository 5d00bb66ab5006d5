"""muon_step over matrices whose last product, which moves the parameters, takes the large kernels: 256, 128 and 64 tiles,
wide, tall and odd sides, each parameter type, float32 parameters with 16-bit copies, gradients of either type.

Tolerances are those of test_gpu_muon.step_check, computed on the GPU in 64 bits.
"""

from __future__ import annotations

import math

import pytest
import torch

import flash_maxsim_amd as fm
from launches import launches
from test_gpu_muon import UNIT, iterate

pytestmark = pytest.mark.gpu

LAST = {256: "muon_next_kernel<3,", 128: ", 2, 2, 4, 4, 2>", 64: ", 2, 2, 2, 2, 4>"}  # of the last product's kernels
SETS = {
    "wide and tall": (256, [(1024, 4096)] * 12 + [(4096, 1024)] * 12),
    "odd": (256, [(1025, 3001), (3001, 1025)] * 2),
    "short and long": (256, [(200, 5000)] * 5 + [(5000, 200)] * 4),
    "two": (128, [(1024, 4096), (4096, 1024)]),
    "one": (128, [(2000, 1500)]),
    "odd, three": (64, [(1003, 517), (517, 1003), (300, 300)]),
}
TYPES = [(torch.bfloat16, torch.bfloat16, None), (torch.float16, torch.float32, None), (torch.float32, torch.float32, None),
         (torch.float32, torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16, torch.float16)]


def inputs(shapes, dtype, grad_dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(s, by):
        return by * torch.randn(s, generator=g, device="cuda")

    return ([n(s, 0.03).to(dtype) for s in shapes], [n(s, 1e-3).to(grad_dtype) for s in shapes], [n(s, 1e-3) for s in shapes])


def check(p0, g, m0, p1, m1, lr, momentum, weight_decay, nesterov, adjust):
    g, m0 = g.double(), m0.double()
    m = momentum * m0 + (1 - momentum) * g
    assert ((m1.double() - m).abs() <= 2.0 ** -22 * (m0.abs() + g.abs())).all()
    u = (1 - momentum) * g + momentum * m if nesterov else m
    o = iterate(u, False)
    tol = 2 * float((iterate(u, True) - o).norm()) + 2.0 ** -16 * float(o.norm())
    r, c = u.shape
    rate = lr * (math.sqrt(max(1.0, r / c)) if adjust == "original" else 0.2 * math.sqrt(max(r, c)))
    p = p0.double() * (1 - lr * weight_decay) - rate * o
    off = float((p1.double() - p).norm())
    assert off <= rate * tol + (UNIT[p0.dtype] + 3 * 2.0 ** -24) * float(p.norm()) + 2.0 ** -22 * rate * float(o.norm()), (r, c)
    # the update itself, not only the sum in which the parameter is the larger: a lost or doubled tile would be as
    # large as the whole of its elements
    moved, want = p1.double() - p0.double() * (1 - lr * weight_decay), -rate * o
    slack = (UNIT[p0.dtype] + 3 * 2.0 ** -24) * p.abs() + 2.0 ** -22 * want.abs()
    lost = ((moved - want).abs() - slack).clamp(min=0)
    for block, size in zip(lost.split(64, 0), want.split(64, 0)):
        for b, s in zip(block.split(64, 1), size.split(64, 1)):
            assert float(b.norm()) <= 0.1 * float(s.norm()) + rate * tol, (r, c)


@pytest.mark.parametrize("dtype,grad_dtype,copy_dtype", TYPES)
@pytest.mark.parametrize("name", SETS)
def test_step(name, dtype, grad_dtype, copy_dtype, tmp_path):
    tile, shapes = SETS[name]
    kw = dict(lr=0.02, momentum=0.95, weight_decay=0.1, nesterov=True, adjust="original")
    if name in ("odd", "one"):
        kw = dict(lr=0.05, momentum=0.9, weight_decay=0.02, nesterov=False, adjust="match_rms_adamw")
    p, g, m = inputs(shapes, dtype, grad_dtype, len(shapes))
    P, M = [t.clone() for t in p], [t.clone() for t in m]
    C = None if copy_dtype is None else [torch.empty(s, device="cuda", dtype=copy_dtype) for s in shapes]
    fm.muon_step(P, g, M, copies=C, **kw)
    for i in range(len(shapes)):
        check(p[i], g[i], m[i], P[i], M[i], **kw)
        assert C is None or torch.equal(C[i], P[i].to(copy_dtype))
    ran = launches(lambda: fm.muon_step(P, g, M, copies=C, **kw), tmp_path)
    assert LAST[tile] in ran[-1][0] and "<3," in ran[-1][0], ran[-1][0]


def test_step_at_any_address():
    """Parameters, gradients, momenta and copies that begin at any element, rows of odd widths."""
    for dtype, copy_dtype in ((torch.bfloat16, None), (torch.float32, torch.bfloat16)):
        for shapes in ([(1025, 3001), (3001, 1025)] * 2, [(1003, 517), (517, 1003)], [(1501, 1999)]):
            p, g, m = inputs(shapes, dtype, torch.bfloat16, 5)

            def odd(t):
                return torch.full((t.numel() + 2,), 7.0, device="cuda", dtype=t.dtype)

            stores = [[odd(t) for t in x] for x in (p, g, m)]
            P, G, M = ([s[1:-1].view(t.shape).copy_(t) for s, t in zip(ss, x)] for ss, x in zip(stores, (p, g, m)))
            C = None
            if copy_dtype:
                stores.append([odd(t.to(copy_dtype)) for t in p])
                C = [s[1:-1].view(t.shape) for s, t in zip(stores[-1], p)]
            fm.muon_step(P, G, M, copies=C)
            aligned = [t.clone() for t in p], [t.clone() for t in m]
            fm.muon_step(aligned[0], g, aligned[1])
            for i in range(len(shapes)):
                assert torch.equal(P[i], aligned[0][i]) and torch.equal(M[i], aligned[1][i])
                assert C is None or torch.equal(C[i], P[i].to(copy_dtype))
            assert all(s[0] == 7 and s[-1] == 7 for ss in stores for s in ss)


def test_alone_and_among_others():
    """A matrix's result does not depend on the tile that the others' number chooses."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for shape in ((1024, 4096), (1003, 517), (700, 900), (3001, 1025)):
        u = torch.randn(shape, generator=g, device="cuda")
        alone = fm.orthogonalize(u)
        for others in (2, 9, 30):
            assert all(torch.equal(o, alone) for o in fm.orthogonalize([u] * others)), (shape, others)


@pytest.mark.parametrize("shapes", [[(301, 60001)], [(60001, 301), (64, 300000)], [(130, 140000), (100, 30)]])
def test_sums_of_squares_over_longer_chunks(shapes):
    """More than 2^24 elements: a workgroup adds up the squares of several chunks, the last one's end early."""
    for dtype, grad_dtype in ((torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)):
        kw = dict(lr=0.02, momentum=0.95, weight_decay=0.1, nesterov=True, adjust="original")
        p, g, m = inputs(shapes, dtype, grad_dtype, 4)
        P, M = [t.clone() for t in p], [t.clone() for t in m]
        fm.muon_step(P, g, M, **kw)
        for i in range(len(shapes)):
            check(p[i], g[i], m[i], P[i], M[i], **kw)
