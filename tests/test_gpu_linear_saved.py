"""What linear keeps for its backward: an operand only where a gradient that needs it is wanted."""

from __future__ import annotations

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_linear import ACTIVATIONS, _LinearFn

pytestmark = pytest.mark.gpu

M, N = 150, 72
NATIVE = fm.linear


def PYTHON(x, w, b, name, r):
    return _LinearFn.apply(x, w, b, ACTIVATIONS[name], r)


def make(K):
    g = torch.Generator().manual_seed(K)
    shapes = {"x": (M, K), "w": (N, K), "b": (N,), "r": (M, N), "dy": (M, N)}
    return {k: (torch.randn(*s, generator=g) * (0.2 if k == "w" else 1)).half().cuda() for k, s in shapes.items()}


def trained(t, leaves):
    return {k: v.clone().requires_grad_(k in leaves) for k, v in t.items()}


# dx reads w, dw reads x, and either and db the slopes
@pytest.mark.parametrize("leaves,needs", [("x", "ws"), ("w", "xs"), ("b", "s"), ("r", ""), ("xw", "xws"), ("xb", "ws"),
                                          ("wbr", "xs"), ("br", "s"), ("xwbr", "xws")])
@pytest.mark.parametrize("name", [None, "silu"])
@pytest.mark.parametrize("K", [96, 77])
@pytest.mark.parametrize("fn", [NATIVE, PYTHON])
def test_only_what_the_gradients_need_is_kept(fn, K, name, leaves, needs):
    t = trained(make(K), leaves)
    kept = []

    def pack(s):
        kept.append("s" if s.dtype == torch.int16 else "w" if s.shape[0] == N else "x")
        return s

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda s: s):
        y = fn(t["x"], t["w"], t["b"], name, t["r"])
    assert sorted(kept) == sorted(c for c in needs if name or c != "s")
    got = torch.autograd.grad(y, [t[k] for k in leaves], t["dy"])
    full = trained(make(K), "xwbr")
    want = dict(zip("xwbr", torch.autograd.grad(NATIVE(*(full[k] for k in "xwb"), name, full["r"]),
                                                [full[k] for k in "xwbr"], t["dy"])))
    assert all(torch.equal(g, want[k]) for g, k in zip(got, leaves))


# torch's linear layer allows each of these changes between the passes
@pytest.mark.parametrize("leaves,changed", [("x", "x"), ("xb", "xr"), ("w", "w"), ("wb", "wr"), ("b", "xw"), ("r", "xwb")])
@pytest.mark.parametrize("name", [None, "gelu"])
@pytest.mark.parametrize("fn", [NATIVE, PYTHON])
def test_operands_changed_before_the_backward(fn, name, leaves, changed):
    t = trained(make(96), leaves)
    want = torch.autograd.grad(fn(t["x"], t["w"], t["b"], name, t["r"]), [t[k] for k in leaves], t["dy"])
    y = fn(t["x"], t["w"], t["b"], name, t["r"])
    with torch.no_grad():
        for k in changed:
            t[k].add_(1.0)
    got = torch.autograd.grad(y, [t[k] for k in leaves], t["dy"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("leaves,changed", [("w", "x"), ("x", "w"), ("xw", "x"), ("xw", "w")])
@pytest.mark.parametrize("fn", [NATIVE, PYTHON])
def test_operands_that_the_backward_reads_must_stay(fn, leaves, changed):
    t = trained(make(96), leaves)
    y = fn(t["x"], t["w"], t["b"], "relu", t["r"])
    with torch.no_grad():
        t[changed].add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, [t[k] for k in leaves], t["dy"])
