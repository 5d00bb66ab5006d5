"""The trained layers together: the head of examples/train_token_head.py in front of MaxSim."""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

import flash_maxsim_amd as fm

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "train_token_head.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_token_head", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("bits", [32, 8])
def test_training_learns(example, bits):
    losses = example.train(steps=25, bits=bits, batch=12, Ld=60, hidden=128, inner=256, d=64)
    assert all(math.isfinite(x) for x in losses)
    # chance is log 12; the head learns to see a query's own document through the noise
    assert sum(losses[-5:]) / 5 < 0.7 * sum(losses[:5]) / 5


def test_head_gradients_reach_every_weight(example):
    """Against the same head and MaxSim in float64 on the CPU. bfloat16 keeps 8 bits and the head has five layers
    with two roundings each, so a gradient is within a tenth of its length."""
    head = example.TokenHead(64, 128, 32, seed=3)
    g = torch.Generator().manual_seed(4)
    hq, hd = torch.randn(3, 8, 64, generator=g).bfloat16(), torch.randn(5, 20, 64, generator=g).bfloat16()
    coef = torch.randn(3, 5, generator=g)
    scores = fm.flash_maxsim_train_batched(head(hq.cuda()), head(hd.cuda()))
    names = list(head.w)
    got = torch.autograd.grad((scores * coef.cuda()).sum(), [head.w[k] for k in names])

    w = {k: v.detach().cpu().double().requires_grad_(True) for k, v in head.w.items()}

    def plain(h):
        x = F.layer_norm(h, (64,), w["norm1.w"], w["norm1.b"])
        x = F.gelu(x @ w["up.w"].t() + w["up.b"]) @ w["down.w"].t() + w["down.b"] + h
        x = F.layer_norm(x, (64,), w["norm2.w"], w["norm2.b"])
        return F.normalize(x @ w["out.w"].t() + w["out.b"], dim=-1)

    q, d = plain(hq.double()), plain(hd.double())
    s = torch.einsum("qik,djk->qdij", q, d).max(-1).values.sum(-1)
    want = torch.autograd.grad((s * coef.double()).sum(), [w[k] for k in names])
    for k, a, b in zip(names, got, want):
        assert (a.cpu().double() - b).norm() <= 0.1 * b.norm() + 1e-6, k
