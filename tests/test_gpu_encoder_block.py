"""The layers of an encoder and its optimizers together: examples/train_encoder_block.py."""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

import flash_maxsim_amd as fm

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "train_encoder_block.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_encoder_block", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_training_runs(example):
    losses = example.train(steps=4, batch=6, Ld=50, vocabulary=300, hidden=64, inner=96, d=32)
    assert len(losses) == 4 and all(math.isfinite(x) for x in losses)


class Rounded(torch.autograd.Function):
    """To bfloat16 and back, in both directions."""

    @staticmethod
    def forward(ctx, t):
        return t.bfloat16().to(t.dtype)

    @staticmethod
    def backward(ctx, g):
        return g.bfloat16().to(g.dtype)


def plain(w, ids, hidden, blocks, r):
    """The encoder in elementary operations, in the type of its weights, r after every operator's result."""
    h = r(w["table"][ids] * math.sqrt(hidden))
    x = r(F.layer_norm(h, (hidden,), w["norm.w"], w["norm.b"]))

    def rms(v):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5)

    for i in range(blocks):
        f = r(F.silu(r(x @ w[f"{i}.gate"].t())) * r(x @ w[f"{i}.up"].t()))
        f = r(f @ w[f"{i}.down"].t())
        h = h + w[f"{i}.scale"] * rms(f) * w[f"{i}.post"]
        x, h = r(rms(h) * w[f"{i}.norm"]), r(h)
    return r(F.normalize(r(x @ w["out.w"].t() + w["out.b"]), dim=-1))


def test_gradients_reach_every_weight(example):
    """Against the same encoder and MaxSim in float64 on the CPU, for the doc tokens that MaxSim takes (the largest of the
    bfloat16 embeddings' products: where two are as good as equal float64 may take the other). How far gradients may be is
    what bfloat16 costs: the same encoder in float64 with every operator's result and gradient rounded is that far, and
    the layers, whose roundings fall elsewhere, may be twice as far."""
    model = example.TokenEncoder(200, 64, 104, 2, 32, seed=3)
    g = torch.Generator().manual_seed(4)
    queries, docs = torch.randint(1, 200, (3, 8), generator=g), torch.randint(1, 200, (5, 20), generator=g)
    docs[2, 15:] = 0
    lengths = torch.tensor([20, 20, 15, 20, 20], dtype=torch.int32)
    coef = torch.randn(3, 5, generator=g)
    q, d = model(queries.cuda()), model(docs.cuda())
    scores = fm.flash_maxsim_train_batched(q, d, lengths.cuda())
    names = list(model.w)
    got = torch.autograd.grad((scores * coef.cuda()).sum(), [model.w[k] for k in names])

    def products(q, d):
        s = torch.einsum("qik,djk->qdij", q, d)
        return s.masked_fill(torch.arange(20) >= lengths[:, None, None], -math.inf)

    taken = products(q.detach().cpu().double(), d.detach().cpu().double()).argmax(-1, keepdim=True)

    def gradients(r):
        w = {k: v.detach().cpu().double().requires_grad_(True) for k, v in model.w.items()}
        s = products(plain(w, queries, 64, 2, r), plain(w, docs, 64, 2, r)).gather(-1, taken).sum((-1, -2))
        return torch.autograd.grad((s * coef.double()).sum(), [w[k] for k in names])

    for k, a, b, c in zip(names, got, gradients(lambda t: t), gradients(Rounded.apply)):
        off, cost = (a.cpu().double() - b).norm(), (c - b).norm()
        assert off <= 2 * cost + 2.0 ** -8 * b.norm(), (k, float(off), float(cost), float(b.norm()))
    assert not got[0][0].any()  # padding


def test_one_block_and_its_step_in_a_graph(example):
    """Forward, backward and both optimizers' steps captured once and replayed, with eager steps of a copy between."""
    def fresh():
        model = example.TokenEncoder(60, 64, 64, 1, 32, seed=5)
        state = [torch.zeros_like(model.master[k]) for k in model.matrices]
        others = [k for k in model.w if k not in model.matrices]
        moments = [fm.adamw_state(model.master[k]) for k in others]
        return model, state, others, moments

    ids = torch.randint(1, 60, (4, 16), generator=torch.Generator().manual_seed(1)).cuda()
    coef = torch.randn(4, 16, 32, generator=torch.Generator().manual_seed(2)).cuda()

    def step(model, state, others, moments):
        names = list(model.w)
        grads = dict(zip(names, torch.autograd.grad((model(ids).float() * coef).sum(), [model.w[k] for k in names])))
        fm.muon_step([model.master[k] for k in model.matrices], [grads[k] for k in model.matrices], state, lr=0.01,
                     copies=[model.w[k] for k in model.matrices])
        fm.adamw_step([model.master[k] for k in others], [grads[k] for k in others], [m for m, _ in moments],
                      [v for _, v in moments], 1, copies=[model.w[k] for k in others])

    captured, eager = fresh(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*captured)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*captured)
    step(*eager)
    for k in range(3):
        ids.copy_(torch.randint(1, 60, (4, 16), generator=torch.Generator().manual_seed(10 + k)))
        graph.replay()
        torch.cuda.synchronize()
        step(*eager)
        for name in captured[0].w:
            assert torch.equal(captured[0].master[name], eager[0].master[name]), name
            assert torch.equal(captured[0].w[name], eager[0].w[name]), name


def test_captured_backward_beside_an_eager_graph():
    """A leaf whose eager graph, built on the default stream, still lives: the captured backward is refused, and works once
    that graph is gone. Gradients that are not wanted do not count."""
    rows = lambda: torch.randn(8, 64, device="cuda", dtype=torch.float16)  # noqa: E731
    x, w, table = rows(), rows(), torch.randn(20, 64, device="cuda")
    ids = torch.randint(0, 20, (8,), device="cuda")
    calls = {"gated": (lambda a, b: fm.gated_linear(a, b, b), rows(), w), "norm": (lambda a, b: fm.residual_norm(a, b)[1], rows(), x),
             "embedding": (lambda a, b: fm.embedding(ids, a), table, w)}
    for name, (call, leaf, other) in calls.items():
        leaf, other = leaf.requires_grad_(True), other.detach().clone().requires_grad_(True)
        dy = torch.ones_like(call(leaf, other))

        def backward(leaf=leaf, call=call, other=other, dy=dy):
            return torch.autograd.grad(call(leaf, other), leaf, dy)[0]

        want = backward()
        eager = call(leaf, other)
        with pytest.raises(RuntimeError, match="still lives"), torch.cuda.graph(torch.cuda.CUDAGraph()):
            backward()
        assert torch.equal(backward(), want), name
        del eager
        only = call(leaf.detach(), other) if name != "embedding" else None  # holds the other's gradient alone
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = backward()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want), name
            assert torch.equal(backward(), want), name
        del only
