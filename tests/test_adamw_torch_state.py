"""AdamW continues the states of torch's AdamW, whose moments are of the parameters' type."""

from __future__ import annotations

import copy

import pytest
import torch

import flash_maxsim_amd as fm


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_moments_of_torchs_states_are_float32(dtype):
    """torch keeps the moments of 16-bit parameters in 16 bits."""
    g = torch.Generator().manual_seed(9)
    a = torch.nn.Parameter(torch.randn(50, 7, generator=g).to(dtype))
    theirs = torch.optim.AdamW([a])
    for _ in range(2):
        a.grad = torch.randn(50, 7, generator=g).to(dtype)
        theirs.step()
    b = torch.nn.Parameter(a.detach().clone())
    mine = fm.AdamW([b])
    mine.load_state_dict(theirs.state_dict())
    for k in ("exp_avg", "exp_avg_sq"):
        want = theirs.state[a][k]
        assert want.dtype == dtype and mine.state[b][k].dtype == torch.float32
        assert torch.equal(mine.state[b][k], want.float())
    assert mine.state[b]["step"] == 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_torchs_16_bit_states_continue(dtype):
    g = torch.Generator().manual_seed(10)
    init, grads = torch.randn(50, 7, generator=g).to(dtype), [torch.randn(50, 7, generator=g).to(dtype) for _ in range(3)]
    a, b = (torch.nn.Parameter(init.cuda()) for _ in range(2))
    theirs = torch.optim.AdamW([a], lr=1e-2, weight_decay=0.1)
    for k in range(2):
        a.grad = grads[k].cuda()
        theirs.step()
    mine = fm.AdamW([b])
    mine.load_state_dict(copy.deepcopy(theirs.state_dict()))
    b.data.copy_(a.data)
    p, gr, m, v = (t.detach().cpu().double() for t in (a, grads[2], theirs.state[a]["exp_avg"], theirs.state[a]["exp_avg_sq"]))
    m, v = 0.9 * m + 0.1 * gr, 0.999 * v + 0.001 * gr * gr
    upd = 1e-2 * (m / (1 - 0.9 ** 3)) / ((v / (1 - 0.999 ** 3)).sqrt() + 1e-8)
    want = p * (1 - 1e-3) - upd
    b.grad = grads[2].cuda()
    mine.step()
    # one rounding to the parameters' type, and a few in float32
    u = 2.0 ** (-11 if dtype == torch.float16 else -8)
    tol = u * want.abs() + 32 * 2.0 ** -24 * (p.abs() + upd.abs()) + 2.0 ** -25
    got, lost = b.detach().cpu().double(), torch.isinf(p)  # torch's step in float16 can end there: eps rounds to zero
    assert lost.sum() < 5 and torch.equal(got[lost], p[lost])
    assert ((got - want).abs() <= tol * 1.01)[~lost].all()
