"""muon_step refuses a grad_scale inside memory that it writes: the scale is read again after the momenta are written."""

from __future__ import annotations

import pytest
import torch

import flash_maxsim_amd as fm

pytestmark = pytest.mark.gpu


def test_scale_within_what_is_written():
    p, g, m = (torch.full((4, 8), v, device="cuda") for v in (1.0, 0.5, 0.25))
    copy = torch.zeros(4, 8, device="cuda", dtype=torch.bfloat16)
    for scale in (p[0, 0], m[3, 7], m.view(-1)[5:6], p.view(-1)[9:10].view(())):
        with pytest.raises(ValueError, match="share"):
            fm.muon_step([p], [g], [m], grad_scale=scale, copies=[copy])
    with pytest.raises(ValueError, match="share"):
        fm.muon_step([p], [g], [m], grad_scale=copy.view(torch.float32)[0, 0], copies=[copy])
    assert (p == 1).all() and (m == 0.25).all() and not copy.any()
    fm.muon_step([p], [g], [m], grad_scale=g[0, 0], copies=[copy])  # beside gradients, which are only read
    assert torch.allclose(m, torch.full_like(m, 0.95 * 0.25 + 0.05 * 0.25), rtol=1e-6) and torch.equal(copy, p.bfloat16())
