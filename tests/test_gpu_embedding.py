"""embedding against a plain implementation in 64 bits, forward and backward.

Tolerances, u the unit roundoff of the table's type: a row is one float32 product (scale as float32: 2^-24 more)
rounded once; a gradient's row of n tokens is a float32 sum, at most n 2^-24 of its terms' magnitudes, times
the scale, rounded once.
"""

from __future__ import annotations

import math

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_embedding import _EmbeddingFn

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: F32}
TYPES = list(UNIT)


def make(T, V, d, dtype, seed, kind="uniform"):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (T,), generator=g)
    if kind == "one":
        ids[:] = V // 2
    if kind == "frequent":  # half of the tokens are two ids, the others fall off
        ids = (torch.rand(T, generator=g).pow(4) * V).long().clamp(max=V - 1)
        ids[torch.rand(T, generator=g) < 0.4] = V - 1
    return ids, torch.randn(V, d, generator=g).to(dtype), torch.randn(T, d, generator=g).to(dtype)


def exact(ids, w, dy, scale, padding=None):
    V, d = w.shape
    flat, rows = ids.flatten(), dy.reshape(-1, d).double()
    keep = (flat >= 0) & (flat < V)
    if padding is not None:
        keep &= flat != padding
    flat, rows = flat[keep], rows[keep]
    dw = torch.zeros(V, d, dtype=torch.float64).index_add_(0, flat, rows) * scale
    size = torch.zeros(V, d, dtype=torch.float64).index_add_(0, flat, rows.abs()) * abs(scale)
    n = torch.bincount(flat, minlength=V)[:, None]
    return dw, F32 * (n + 3) * size


def check(name, got, want, err):
    got = got.detach().cpu()
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    tol = UNIT[got.dtype] * (want.abs() + err) + err + tiny
    off = (got.double() - want).abs()
    assert got.shape == want.shape
    assert (off <= tol * 1.01).all(), f"{name}: off by up to {off.max().item()}"


def run(ids, w, dy, scale=1.0, padding=None, fn=None):
    ids, w, dy = ids.cuda(), w.cuda().requires_grad_(True), dy.cuda()
    y = fm.embedding(ids, w, scale, padding) if fn is None else fn(ids, w, scale, -1 if padding is None else padding)
    return y, torch.autograd.grad(y, w, dy)[0]


def verify(ids, w, dy, scale=1.0, padding=None):
    y, dw = run(ids, w, dy, scale, padding)
    check("y", y, w[ids].double() * scale, 2 * F32 * (w[ids].double() * scale).abs())
    check("dw", dw, *exact(ids, w, dy, scale, padding))
    assert torch.equal(fm.embedding(ids.cuda(), w.cuda(), scale, padding), y)  # without autograd
    return y, dw


# tokens around the stretches of 32 and the sorts' limits, ids around digits' limits, widths around the pieces
SIZES = [(1, 1, 1), (1, 5, 3), (2, 300, 8), (31, 7, 9), (32, 7, 16), (33, 2, 64), (64, 1000, 100), (65, 3, 513), (200, 50, 1030),
         (1000, 1023, 24), (1025, 1024, 40), (3000, 1025, 77), (5001, 1009, 300), (14336, 70, 33), (14337, 70, 33), (16384, 70, 33), (16385, 70, 33),
         (16400, 1, 8), (20000, 1024, 17), (20480, 100000, 8), (30001, 1048576, 3), (70000, 4097, 64)]


@pytest.mark.parametrize("kind", ["uniform", "frequent", "one"])
@pytest.mark.parametrize("T,V,d", SIZES)
def test_sizes(T, V, d, kind):
    for dtype in TYPES if T < 5000 else [TYPES[(T + d) % 3]]:
        verify(*make(T, V, d, dtype, T + V + d, kind), scale=math.sqrt(d))


@pytest.mark.parametrize("dtype", TYPES)
def test_wide_rows(dtype):
    verify(*make(100, 20, 5000, dtype, 1, "frequent"), scale=0.5)
    verify(*make(40, 9, 65536, dtype, 2), scale=-1.0)


def test_more_ids_than_two_digits():
    ids, w, dy = make(40000, 3000000, 2, torch.float32, 3)
    verify(ids, w, dy)


def test_int32_ids_shapes_and_strides():
    ids, w, dy = make(120, 30, 40, torch.float16, 4)
    want, err = exact(ids, w, dy, 2.0)
    for t in (ids.int(), ids):
        y, dw = run(t.view(2, 3, 20), w, dy.view(2, 3, 20, 40), 2.0)
        assert y.shape == (2, 3, 20, 40)
        check("dw", dw, want, err)
    wide = torch.full((120, 90), 7, dtype=torch.int64)
    wide[:, ::3][:, 5] = ids
    y, dw = run(wide[:, 15], w, dy.t().contiguous().t(), 2.0)
    check("dw", dw, want, err)
    # a table beside others, its rows from any element on; columns first
    store = torch.full((30, 67), float("nan"), dtype=torch.float16, device="cuda")
    store[:, 5:45] = w.cuda()
    for view in (store[:, 5:45], w.cuda().t().contiguous().t()):
        leaf = view.detach().requires_grad_(True)
        y = fm.embedding(ids.cuda(), leaf, 2.0)
        check("y", y, w[ids].double() * 2, 0 * w[ids].double())
        check("dw", torch.autograd.grad(y, leaf, dy.cuda())[0], want, err)
    one = w[:1].cuda().requires_grad_(True)  # one row for all ids
    y = fm.embedding(ids.cuda(), one.expand(30, 40), 2.0)
    (dw,) = torch.autograd.grad(y, one, dy.cuda())
    total = want.sum(0, keepdim=True)
    tol = (err + UNIT[torch.float16] * want.abs()).sum(0) * 1.01 + 32 * UNIT[torch.float16] * want.abs().sum(0)
    assert ((dw.cpu().double() - total).abs() <= tol).all()
    scalar, w1 = torch.tensor(7), w.cuda()
    assert torch.equal(fm.embedding(scalar.cuda(), w1), w1[7])


def test_padding():
    for T in (50, 17000):
        ids, w, dy = make(T, 40, 24, torch.bfloat16, 5, "frequent")
        for padding in (0, 39, int(ids[0])):
            y, dw = verify(ids, w, dy, 1.5, padding)
            assert not dw[padding].any()


def test_ids_outside_the_table():
    for T in (60, 18000):
        ids, w, dy = make(T, 33, 20, torch.float32, 6)
        ids[::7], ids[3::11], ids[5] = -1, 33, 1 << 40
        out = (ids < 0) | (ids >= 33)
        y, dw = run(ids, w, dy)
        assert torch.isnan(y[out.cuda()]).all() and torch.equal(y[~out.cuda()].cpu(), w[ids[~out]])
        check("dw", dw, *exact(ids, w, dy, 1.0))
        none, _, _ = make(T, 33, 20, torch.float32, 6)
        none[:] = -5
        y, dw = run(none, w, dy)
        assert torch.isnan(y).all() and not dw.any()


def test_no_tokens():
    for shape in ((0,), (3, 0)):
        w = torch.randn(700, 24, device="cuda", dtype=torch.float16, requires_grad=True)
        y = fm.embedding(torch.empty(shape, dtype=torch.int64, device="cuda"), w)
        torch.full((700 * 24,), float("nan"), device="cuda", dtype=torch.float16)  # freed: what dw may get holds no zeros
        (dw,) = torch.autograd.grad(y, w, torch.empty(*shape, 24, device="cuda", dtype=torch.float16))
        assert y.shape == (*shape, 24) and dw.shape == w.shape and not dw.any()


def test_values_that_are_not_finite_stay_in_their_row():
    ids, w, dy = make(500, 40, 24, torch.bfloat16, 7)
    dy[100, 3], dy[200, 5] = float("nan"), float("inf")
    _, dw = run(ids, w, dy)
    bad = (~torch.isfinite(dw)).any(1).nonzero().flatten().tolist()
    assert set(bad) == {int(ids[100]), int(ids[200])}


def test_gradient_against_differences():
    ids, w, dy = make(90, 13, 11, torch.float32, 8)
    _, dw = run(ids, w, dy, 3.0)
    d = torch.randn(13, 11, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    h = 1e-5
    f = lambda w: ((w[ids] * 3.0) * dy.double()).sum()  # noqa: E731
    diff = (f(w.double() + h * d) - f(w.double() - h * d)) / (2 * h)
    mine = dw.cpu().double() * d
    assert abs(mine.sum() - diff) <= 1e-5 * mine.abs().sum()


def test_both_paths_agree_and_repeat_bit_for_bit():
    for T in (900, 40000):
        ids, w, dy = make(T, 200, 72, torch.bfloat16, 9, "frequent")
        a, b, c = run(ids, w, dy, 2.0, 3), run(ids, w, dy, 2.0, 3), run(ids, w, dy, 2.0, 3, _EmbeddingFn.apply)
        assert all(torch.equal(x, y) for o in (b, c) for x, y in zip(a, o))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b = run(ids, w, dy, 2.0, 3)
        side.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_order_of_tokens_does_not_reach_other_ids():
    """A row's sum does not depend on where its tokens lie among others."""
    ids, w, dy = make(3000, 50, 16, torch.float32, 10)
    _, dw = run(ids, w, dy)
    other = ids.clone()
    other[ids == 7] = 9  # other ids move; id 20's tokens stay in their order
    _, dw2 = run(other, w, dy)
    want, err = exact(other, w, dy, 1.0)
    check("dw", dw2, want, err)
    assert not dw2[7].any()


@pytest.mark.parametrize("T", [32, 700, 20000])
def test_graph_replays(T):
    """Forward and backward in one graph, replayed with eager calls between."""
    ids, w, dy = (t.cuda() for t in make(T, 500, 40, torch.float16, 12))
    w.requires_grad_(True)

    def step():
        y = fm.embedding(ids, w, 2.0)
        return [y.detach(), torch.autograd.grad(y, w, dy)[0]]

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
        ids.copy_(make(T, 500, 40, torch.float16, 40 + seed, "frequent")[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


HOOKS = [(lambda t: t.cpu(), lambda t: t.cuda()), (lambda t: t, lambda t: t.clone()),
         (lambda t: t, lambda t: torch.stack([t, t], -1)[..., 0])]


@pytest.mark.parametrize("pack,unpack", HOOKS)
def test_saved_tensors_in_another_layout(pack, unpack):
    ids, w, dy = make(300, 40, 24, torch.float16, 14)
    for fn in (None, _EmbeddingFn.apply):
        want = run(ids, w, dy, fn=fn)
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            got = run(ids, w, dy, fn=fn)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_changed_ids_and_second_derivatives():
    ids, w, dy = (t.cuda() for t in make(30, 8, 16, torch.float32, 15))
    w.requires_grad_(True)
    y = fm.embedding(ids, w)
    first = torch.autograd.grad(y, w, dy, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(y, w, dy, retain_graph=True)[0])
    ids.add_(0)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, w, dy)
    (dw,) = torch.autograd.grad(fm.embedding(ids, w).square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        dw.square().sum().backward()


def test_views_read_with_their_sign():
    ids, w, dy = (t.cuda() for t in make(30, 24, 40, torch.float16, 6))
    got, want = [], []
    for out, f in ((got, torch._neg_view), (want, lambda t: -t)):
        leaf = f(w).detach().requires_grad_(True)
        y = fm.embedding(ids, leaf, 3.0)
        out += [y, torch.autograd.grad(y, leaf, f(dy))[0], fm.embedding(f(-ids), w, 3.0)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    w = torch.zeros(10, 8, device="cuda")
    ids = torch.zeros(4, device="cuda", dtype=torch.int64)
    for bad in (dict(ids=ids.float()), dict(ids=ids.short()), dict(weight=w.double())):
        with pytest.raises(TypeError):
            fm.embedding(**({"ids": ids, "weight": w} | bad))
    for bad in (dict(scale=float("inf")), dict(padding_idx=10), dict(padding_idx=-1)):
        with pytest.raises(ValueError):
            fm.embedding(ids, w, **bad)
    for bad in (w[0], w[:0], w[:, :0]):
        with pytest.raises(AssertionError):
            fm.embedding(ids, bad)
    for a, b in ((ids.cpu(), w), (ids, w.cpu())):
        with pytest.raises(RuntimeError):
            fm.embedding(a, b)
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(w, w)
        with pytest.raises(NotImplementedError):
            fm.embedding(ids, t)
        inside = fm.embedding(ids, w)
    assert torch.equal(inside, fm.embedding(ids, w))
