"""embedding's gradient where a bound over all of an id's tokens says little: ids of very many tokens.

Whole numbers: their float32 sums are exact up to 2^24 whatever their order, so the gradient has to equal the rounded
sum, and a stretch of tokens, a partial sum or a wave of the join that is left out or taken twice shows. And values of any
kind, by the order in which the kernels add: a stretch of at most 32 terms, then up to 25 partial sums one after the other,
or every sixteenth of them and the sixteen: 2^-24 (32 + max(25, n / 512 + 16) + 3) of the terms' magnitudes.
"""

from __future__ import annotations

import pytest
import torch

import flash_maxsim_amd as fm
from launches import launches
from test_gpu_embedding import F32, SIZES, TYPES, UNIT, make, run

pytestmark = pytest.mark.gpu

MORE = [(100, 3, 40), (800, 2, 24), (801, 2, 24), (832, 1, 24), (833, 1, 24), (4097, 2, 9), (150000, 3, 72), (400000, 5000, 20)]


def whole(ids, V, d, dtype, seed):
    """dy of whole numbers, and the sums."""
    dy = torch.randint(-16, 17, (len(ids), d), generator=torch.Generator().manual_seed(seed)).to(dtype)
    dw = torch.zeros(V, d, dtype=torch.int64).index_add_(0, ids, dy.long())
    assert dw.abs().max() < 1 << 22
    return dy, dw


@pytest.mark.parametrize("kind", ["uniform", "frequent", "one"])
@pytest.mark.parametrize("T,V,d", SIZES + MORE)
def test_whole_numbers(T, V, d, kind):
    for dtype in TYPES if T < 5000 else [torch.float32, TYPES[T % 2]]:
        ids, w, _ = make(T, V, d, dtype, T + V + d, kind)
        dy, dw = whole(ids, V, d, dtype, T + d)
        for scale in (1.0, -0.25):
            want = (dw.double() * scale).to(dtype)
            assert torch.equal(run(ids, w, dy, scale)[1].cpu(), want), (dtype, scale)


@pytest.mark.parametrize("T,padding", [(900, 1), (20000, 0), (150000, 1)])
def test_whole_numbers_with_padding_and_ids_outside(T, padding):
    """The padding id has half of the tokens."""
    ids = torch.randint(-1, 4, (T,), generator=torch.Generator().manual_seed(T))
    ids[:: 2] = padding
    keep = (ids >= 0) & (ids < 3) & (ids != padding)
    dy, _ = whole(ids.clamp(0, 3), 4, 40, torch.float32, T)
    want = torch.zeros(3, 40).index_add_(0, ids[keep], dy[keep])
    assert torch.equal(run(ids, torch.zeros(3, 40), dy, 1.0, padding)[1].cpu(), want)


@pytest.mark.parametrize("T,V,d", [(3000, 2, 24), (14336, 1, 33), (20000, 1024, 17), (70000, 4097, 64), (150000, 3, 72)])
def test_any_values_by_the_order_of_the_sums(T, V, d):
    for kind in ("uniform", "frequent", "one"):
        for dtype in TYPES:
            ids, w, dy = make(T, V, d, dtype, T + d, kind)
            got = run(ids, w, dy, 0.5)[1].cpu().double()
            want = torch.zeros(V, d, dtype=torch.float64).index_add_(0, ids, dy.double()) * 0.5
            size = torch.zeros(V, d, dtype=torch.float64).index_add_(0, ids, dy.double().abs()) * 0.5
            n = torch.bincount(ids, minlength=V)[:, None]
            err = F32 * (32 + (n / 512 + 16).clamp(min=25) + 3) * size
            tol = UNIT[dtype] * (want.abs() + err) + err + 2.0 ** -25
            assert ((got - want).abs() <= tol * 1.01).all(), (kind, dtype, ((got - want).abs() / tol).max())


@pytest.mark.parametrize("T", [9, 5000, 40000])
@pytest.mark.parametrize("d,dtype", [(601, torch.float16), (299, torch.float32), (608, torch.bfloat16)])
def test_whole_numbers_past_the_caches(T, d, dtype):
    V = 200003
    g = torch.Generator(device="cuda").manual_seed(T + d)
    ids = torch.randint(V - 20000, V, (T,), generator=g, device="cuda")
    ids[: T // 3] = 7
    dy = torch.randint(-16, 17, (T, d), generator=g, device="cuda").to(dtype)
    want = torch.zeros(V, d, dtype=torch.float32, device="cuda").index_add_(0, ids, dy.float())  # exact, below 2^24
    assert want.abs().max() < 1 << 22
    assert torch.equal(run(ids, torch.zeros(V, d, dtype=dtype), dy)[1], want.to(dtype))


@pytest.mark.parametrize("T,V,d,padding", [(262144, 1000, 8, None), (262145, 1000, 8, 3), (262145, 1, 5, None), (300001, 2, 4, 1),
                                           (700000, 100000, 4, 7), (1000003, 3000000, 2, None), (4500000, 40, 2, 39)])
def test_whole_numbers_of_many_tokens(T, V, d, padding):
    """Around the count of tokens from which digits are added up in a launch of their own, one to three digits."""
    ids = make(T, V, d, torch.float32, T + V, "frequent")[0]
    dy = torch.randint(-4, 5, (T, d), generator=torch.Generator().manual_seed(T)).float()
    keep = ids >= 0 if padding is None else ids != padding
    want = torch.zeros(V, d, dtype=torch.int64).index_add_(0, ids[keep], dy[keep].long())
    assert want.abs().max() < 1 << 22
    assert torch.equal(run(ids, torch.zeros(V, d), dy, 1.0, padding)[1].cpu().long(), want)


def test_digits_of_many_tokens_are_added_up_once(tmp_path):
    """Not by every workgroup of a pass for itself: a launch in each of the two passes."""
    for T, times in ((262144, 0), (262145, 2)):
        ids, w = torch.arange(T, device="cuda") % 5000, torch.zeros(5000, 4, device="cuda", requires_grad=True)
        dy = torch.ones(T, 4, device="cuda")
        ran = launches(lambda: torch.autograd.grad(fm.embedding(ids, w), w, dy), tmp_path)
        assert sum("embedding_scan_kernel" in name for name, _ in ran) == times
