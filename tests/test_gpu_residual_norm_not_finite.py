"""residual_norm of rows that are not finite, element by element against the formula in 64 bits.

Where the formula gives an infinity or NaN the kernels give the same one, whichever column of a row it comes from:
rows of odd widths have columns that two lanes hold. A bad row's finite values are of few float32 operations
(h of two products and a sum, y of a product with zero and a sum): 4 x 2^-24 of their terms, and rounded once. Rows
and column sums besides are bounded as in test_gpu_residual_norm.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_residual_norm import F32, ROWS, TYPES, UNIT, VECTORS, call, exact, make, run

pytestmark = pytest.mark.gpu

BAD = 3  # the row


def columns(d, dtype):
    """One that only one lane holds, the first and the last that two hold, and the row's last."""
    piece = 4 if dtype == torch.float32 else 8
    rest = d % piece
    return sorted({d // 3, d - piece, d - rest - 1, d - 1}) if rest else [d // 3, d - 1]


def same(name, got, want, tol):
    got = got.detach().cpu().double()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]), name
    off = (got - want).abs()[finite]
    assert (off <= tol[finite]).all(), (name, off.max())


def verify(s, got):
    want, err = exact(s)
    alpha_r = (s["alpha"] * s["r"].double()).abs()
    terms = {"h": want["h"].abs() + 2 * alpha_r, "y": want["y"].abs()}
    for n, v in got.items():
        u = UNIT[v.dtype]
        tol = u * (want[n].abs() + err[n]) + err[n] + (2.0 ** -25 if v.dtype == torch.float16 else 0.0)
        if want[n].ndim == 2 and n in terms:
            few = u * want[n].abs() + 4 * F32 * terms[n] + 2.0 ** -25
            tol = torch.where(torch.isfinite(err[n]), tol, few)  # of a row whose bound is not finite
        same(n, v, want[n], tol * 1.01)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [9, 40, 515, 771, 1023, 1025, 2050, 3001, 4101, 8191])
def test_an_infinity_in_any_column(d, dtype, norm):
    for parts in ((), ("post", "scale")):
        for column in columns(d, dtype):
            for name in ("x", "r"):
                s = make(6, d, dtype, d, parts, norm)
                s[name][BAD, column] = float("inf")
                h, y = call({k: None if s[k] is None else s[k].cuda() for k in ROWS + VECTORS}, s)
                verify(s, {"h": h, "y": y})


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [9, 40, 515, 771, 1023, 1025, 2050, 3001, 4101, 8191])
def test_an_infinity_among_the_gradients(d, dtype, norm):
    """Of y's gradient, which the row's sums take: dr is not finite anywhere in the row, by the formula's signs."""
    for parts in ((), ("post", "scale")):
        for column in columns(d, dtype):
            s = make(6, d, dtype, d + 1, parts, norm)
            s["dy"][BAD, column] = float("inf")
            verify(s, run(s))
