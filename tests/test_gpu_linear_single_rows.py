"""Operands of one row or none, whose row strides say nothing: any is taken."""

from __future__ import annotations

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_linear import ACTIVATIONS, _LinearFn

pytestmark = pytest.mark.gpu


def inside(t, width):
    """t as the first columns of a buffer of `width` elements a row."""
    wide = torch.full((t.shape[0], width), float("nan"), dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


@pytest.mark.parametrize("width", [178, 168, (1 << 22) + 8])
@pytest.mark.parametrize("M,N", [(1, 24), (9, 1), (1, 1), (0, 24), (0, 1)])
@pytest.mark.parametrize("K", [168, 163])
@pytest.mark.parametrize("transposed", [False, True])
def test_any_stride_of_a_single_row(transposed, K, M, N, width):
    g = torch.Generator().manual_seed(M + N)
    x, w, r, dy = (torch.randn(*s, generator=g).half().cuda() for s in ((M, K), (N, K), (M, N), (M, N)))

    def run(x, w, r, dy, fn):
        x, w, r = (t.detach().requires_grad_(True) for t in (x, w, r))
        y = fn(x, w, None, "gelu", r)
        return [y.detach(), *torch.autograd.grad(y, (x, w, r), dy)]

    want = run(x, w, r, dy, fm.linear)
    # the other operand by columns: the call takes the Python path
    xs = x.t().contiguous().t() if transposed and M > 1 else inside(x, width) if M < 2 else x
    ws = w.t().contiguous().t() if transposed and N > 1 else inside(w, width) if N < 2 else w
    for fn in (fm.linear, lambda x, w, b, a, r: _LinearFn.apply(x, w, b, ACTIVATIONS[a], r)):
        got = run(xs, ws, inside(r, N + 3), inside(dy, N + 5), fn)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
