"""embedding with padding_idx by the native host path: the same results as the Python path's, the same refusals."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_embedding import _EmbeddingFn
from test_gpu_embedding import check, exact, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 40, 900, 20000])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_padding_takes_the_native_path(T, dtype):
    ids, w, dy = make(T, 50, 24, dtype, T, "frequent")
    for padding in (0, 49, int(ids[0])):
        leaf = w.cuda().requires_grad_(True)
        y = fm.embedding(ids.cuda(), leaf, 1.5, padding)
        assert y.grad_fn.name() == "FlashMaxSimEmbeddingBackward"
        (dw,) = torch.autograd.grad(y, leaf, dy.cuda())
        check("dw", dw, *exact(ids, w, dy, 1.5, padding))
        assert not dw[padding].any()
        other = _EmbeddingFn.apply(ids.cuda(), leaf, 1.5, padding)
        assert torch.equal(y, other) and torch.equal(dw, torch.autograd.grad(other, leaf, dy.cuda())[0])
        assert torch.equal(fm.embedding(ids.cuda(), leaf.detach(), 1.5, padding), y)
    assert torch.equal(fm.embedding(ids.cuda(), w.cuda(), 1.5, np.int64(3)), y)  # another kind of number


def test_refusals():
    w, ids = torch.zeros(10, 8, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.int64)
    for bad in (-1, -2, 10, 1 << 62, 1 << 70, -(1 << 70)):
        with pytest.raises(ValueError, match="padding_idx"):
            fm.embedding(ids, w, padding_idx=bad)
