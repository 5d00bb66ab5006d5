"""A backward pass captured into a graph beside a living eager graph of the same leaf that was built on the default
stream: refused by every layer's node, native or in Python, and sound once that graph is gone."""

from __future__ import annotations

import pytest
import torch

import flash_maxsim_amd as fm
from flash_maxsim_amd.flash_maxsim_embedding import _EmbeddingFn
from flash_maxsim_amd.flash_maxsim_gated import _GatedLinearFn
from flash_maxsim_amd.flash_maxsim_linear import _LinearFn
from flash_maxsim_amd.flash_maxsim_norm import _LayerNormFn
from flash_maxsim_amd.flash_maxsim_residual_norm import _ResidualNormFn

pytestmark = pytest.mark.gpu


def rows(*shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(sum(shape))).cuda().half()


def layers(x, r, w, u, out, q, docs, ids):
    """name: (call of the leaf, the leaf's like). x and r [8, 64], w and u [16, 64], out [8, 16], q [6, 64], docs [3, 12, 64]"""
    return {
        "linear": (lambda a: fm.linear(a, w), x),
        "linear, its weight": (lambda a: fm.linear(x, a, activation="gelu"), w),
        "linear, its bias": (lambda a: fm.linear(x, w, a), out[0]),
        "linear, its residual": (lambda a: fm.linear(x, w, residual=a), out),
        "layer_norm": (lambda a: fm.layer_norm(a), x),
        "layer_norm, its weight": (lambda a: fm.layer_norm(x, a), x[0]),
        "gated_linear": (lambda a: fm.gated_linear(a, w, u), x),
        "gated_linear, a weight": (lambda a: fm.gated_linear(x, w, a), u),
        "residual_norm": (lambda a: fm.residual_norm(a, r)[1], x),
        "residual_norm, its scale": (lambda a: fm.residual_norm(x, r, scale=a)[0], x[0]),
        "embedding": (lambda a: fm.embedding(ids, a), w),
        "embedding with padding": (lambda a: fm.embedding(ids, a, padding_idx=0), w),
        "train, its query": (lambda a: fm.flash_maxsim_train(a, docs), q),
        "train, its docs": (lambda a: fm.flash_maxsim_train(q, a), docs),
        "train_batched": (lambda a: fm.flash_maxsim_train_batched(a, docs), q[None]),
        "linear in Python": (lambda a: _LinearFn.apply(a, w, None, 0, None), x),
        "layer_norm in Python": (lambda a: _LayerNormFn.apply(a, None, None, 1e-5), x),
        "gated_linear in Python": (lambda a: _GatedLinearFn.apply(a, w, u, None, None, 4), x),
        "residual_norm in Python": (lambda a: _ResidualNormFn.apply(a, r, *[None] * 6, False, 1.0, 0, 1e-5)[0], x),
        "embedding in Python": (lambda a: _EmbeddingFn.apply(ids, a, 1.0, 0), w),
    }


NAMES = list(layers(*[torch.zeros(1, 1)] * 8))


@pytest.mark.parametrize("name", NAMES)
def test_refused_while_the_eager_graph_lives(name):
    operands = rows(8, 64), rows(8, 64) + 1, rows(16, 64), rows(16, 64) - 1, rows(8, 16), rows(6, 64), rows(3, 12, 64)
    call, like = layers(*operands, torch.arange(8, device="cuda") % 5)[name]
    leaf = like.clone().requires_grad_(True)
    dy = torch.ones_like(call(leaf))

    def backward():
        return torch.autograd.grad(call(leaf), leaf, dy)[0]

    want = backward()
    eager = call(leaf)
    with pytest.raises(RuntimeError, match="still lives"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        backward()
    assert torch.equal(torch.autograd.grad(eager, leaf, dy)[0], want)  # the eager graph itself goes on
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = backward()
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert torch.equal(backward(), want)
