"""AdamW's state: what deep copies and pickles keep."""

from __future__ import annotations

import copy
import io
import pickle

import pytest
import torch

import flash_maxsim_amd as fm


def made(device, bits, copies):
    g = torch.Generator().manual_seed(3)
    ps = [torch.nn.Parameter(torch.randn(n, generator=g).to(device)) for n in (300, 7, 64)]
    cs = [None if i == 1 else p.detach().bfloat16() for i, p in enumerate(ps)] if copies else None
    return fm.AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 5e-3}], lr=1e-2, state_bits=bits, copies=cs)


def params(opt):
    return [p for g in opt.param_groups for p in g["params"]]


def copies_of(opt):
    return [opt._copies.get(id(p)) for p in params(opt)]


def through_pickle(opt):
    return pickle.loads(pickle.dumps(opt))


def through_file(opt):
    f = io.BytesIO()
    torch.save(opt, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


COPIERS = [copy.deepcopy, through_pickle, through_file]


@pytest.mark.parametrize("again", COPIERS)
@pytest.mark.parametrize("copies", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_copied_optimizers_keep_bits_and_copies(again, copies, bits):
    opt = made("cpu", bits, copies)
    for other in (again(opt), again(again(opt))):
        assert other._bits == bits and len(other._copies) == (2 if copies else 0)
        for p, q, c, e in zip(params(opt), params(other), copies_of(opt), copies_of(other)):
            assert p is not q and torch.equal(p, q) and (c is None) == (e is None)
            assert c is None or (c is not e and torch.equal(c, e) and c.dtype == e.dtype)
    assert len(opt._copies) == (2 if copies else 0)
    other = copy.copy(opt)
    assert all(a is b for a, b in zip(copies_of(other), copies_of(opt))) and other._bits == bits


def test_a_copy_of_a_program_keeps_its_tensors_together():
    opt = made("cpu", 32, True)
    ps, cs = params(opt), copies_of(opt)
    opt2, ps2, cs2 = copy.deepcopy((opt, ps, cs))
    assert all(a is b for a, b in zip(params(opt2), ps2)) and all(a is b for a, b in zip(copies_of(opt2), cs2))


@pytest.mark.gpu
@pytest.mark.parametrize("again", COPIERS)
@pytest.mark.parametrize("bits", [32, 8])
def test_copied_optimizers_step_alike(again, bits):
    opt = made("cuda", bits, True)
    g = torch.Generator().manual_seed(4)
    grads = [[torch.randn(p.shape, generator=g).cuda() for p in params(opt)] for _ in range(3)]

    def steps(o, which):
        for k in which:
            for p, t in zip(params(o), grads[k]):
                p.grad = t.clone()
            o.step()

    steps(opt, [0])
    other = again(opt)
    steps(opt, [1, 2])
    steps(other, [1, 2])
    for p, q, c, e in zip(params(opt), params(other), copies_of(opt), copies_of(other)):
        assert p is not q and torch.equal(p, q)
        assert c is None or (torch.equal(e, q.detach().bfloat16()) and torch.equal(c, e) and c is not e)


@pytest.mark.gpu
def test_moments_of_both_kinds_at_one_step():
    """A loaded 32-bit state beside parameters whose moments begin in 8 bits."""
    g = torch.Generator().manual_seed(11)
    init = [torch.randn(40, generator=g).cuda() for _ in range(2)]
    grads = [torch.randn(40, generator=g).cuda() for _ in range(2)]

    def step(opt, ps, which):
        for i, p in enumerate(ps):
            p.grad = grads[i].clone() if i in which else None
        opt.step()

    old = [torch.nn.Parameter(t.clone()) for t in init]
    saved = fm.AdamW(old, state_bits=32)
    step(saved, old, {0})
    ps = [torch.nn.Parameter(t.detach().clone()) for t in old]
    opt = fm.AdamW(ps, state_bits=8)
    opt.load_state_dict(saved.state_dict())
    step(opt, ps, {1})  # now both stand at one step, of 32 and of 8 bits
    step(opt, ps, {0, 1})
    assert opt.state[ps[0]]["exp_avg"].dtype == torch.float32 and opt.state[ps[1]]["exp_avg"].dtype == torch.int8
    step(saved, old, {0})
    assert torch.equal(old[0], ps[0]) and opt.state[ps[1]]["step"] == 2
