"""8-bit moments of blocks with a value that is not finite."""

from __future__ import annotations

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_optim import BLOCK

pytestmark = pytest.mark.gpu


# of 2e19 the square is past float32's range; it stands for a gradient that is itself finite
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), 2e19, -3e38])
@pytest.mark.parametrize("at", [0, 131, BLOCK - 1])
def test_a_block_with_such_a_value_decodes_to_nan(value, at):
    n = 3 * BLOCK + 5
    g = torch.linspace(-1, 1, n)
    g[BLOCK + 7] = 0.0
    g[BLOCK + at] = value
    P, G = torch.ones(n).cuda(), g.cuda()
    m, v = fm.adamw_state(P, 8)
    fm.adamw_step([P], [G], [m], [v], 1, lr=0.1, weight_decay=0.0)
    md, vd = fm.dequantize_adamw(m).cpu(), fm.dequantize_adamw(v).cpu()
    lost = torch.zeros(n, dtype=torch.bool)
    lost[BLOCK:2 * BLOCK] = True
    assert torch.isnan(vd[lost]).all() and torch.isfinite(vd[~lost]).all()
    finite = abs(value) < 3.4e38  # of a finite gradient the first moment is finite
    assert (torch.isfinite(md[lost]).all() if finite else torch.isnan(md[lost]).all()) and torch.isfinite(md[~lost]).all()
    # the next step shows it: all of the block's parameters are NaN, none of the others
    before = P.clone()
    fm.adamw_step([P], [torch.ones_like(P)], [m], [v], 2, lr=0.1, weight_decay=0.0)
    P = P.cpu()
    assert torch.isnan(P[lost]).all() and torch.isfinite(P[~lost]).all() and (P[~lost] != before.cpu()[~lost]).any()
    # and it stays so
    assert torch.isnan(fm.dequantize_adamw(v).cpu()[lost]).all()
