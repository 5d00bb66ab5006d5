"""Queries and docs of one token that lie in wider buffers, through the Python path (int64 lengths)."""

from __future__ import annotations

import pytest
import torch

import flash_maxsim_amd as fm

pytestmark = pytest.mark.gpu


def inside(t, width):
    wide = torch.full((*t.shape[:-1], width), float("nan"), dtype=t.dtype, device=t.device)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


@pytest.mark.parametrize("B,Lq,Ld", [(50, 1, 30), (1, 1, 1), (1, 7, 1), (50, 7, 1), (0, 1, 30)])
@pytest.mark.parametrize("d", [128, 100])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_any_stride_of_a_single_row(dtype, d, B, Lq, Ld):
    g = torch.Generator().manual_seed(B + Lq + d)
    q, docs = torch.randn(Lq, d, generator=g).to(dtype).cuda(), torch.randn(B, Ld, d, generator=g).to(dtype).cuda()
    lengths = torch.full((B,), Ld, device="cuda")
    want = fm.flash_maxsim(q, docs, lengths.int())
    assert torch.equal(fm.flash_maxsim(inside(q, d + 10), inside(docs, d + 10), lengths), want)
    assert torch.equal(fm.flash_maxsim_batched(inside(q[None], d + 10), inside(docs, d + 10), lengths)[0], want)
