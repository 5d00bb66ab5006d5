"""The slopes that linear keeps between its passes, near one and far out where they vanish.

The kernel's own slope: GELU's normal distribution function is the formula of Abramowitz and Stegun 7.1.26, whose
distance from the true one is taken from that formula in 64 bits; every other term is a product of a few float32
factors, and an exponential of an argument q is off by |q| 2^-23 of itself. A slope is held in 16 bits by a code that
does not decrease, so what comes back lies between the codes of the smallest and the largest slope that this allows.
"""

from __future__ import annotations

import math

import pytest
import torch

import flash_maxsim_amd as fm

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
SMOOTH = ["gelu", "gelu_tanh", "silu"]
TYPES = [torch.float16, torch.bfloat16]


def slope(z, name):
    """(slope, its distance in float32, its own slope) of each argument, in 64 bits."""
    if name == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2))
        d = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        x = z.abs() / math.sqrt(2)
        t = 1 / (1 + 0.3275911 * x)
        tail = 0.5 * torch.exp(-x * x) * t * (0.254829592 + t * (-0.284496736 + t * (1.421413741 + t * (
            -1.453152027 + t * 1.061405429))))
        off = (tail - 0.5 * torch.erfc(x)).abs() + (z * z / 2 + 24) * 2 * F32 * (tail + (z * d).abs()) + F32 * p
        return p + z * d, off, d * (2 - z * z)
    if name == "silu":
        s = torch.sigmoid(z)
        off = (z.abs() * 1.5 + 16) * 2 * F32 * (s + z.abs() * s * (1 - s))
        return s * (1 + z * (1 - s)), off, s * (1 - s) * (2 + z * (1 - 2 * s))
    k = 2 * math.sqrt(2 / math.pi)
    q, dq, ddq = k * (z + 0.044715 * z ** 3), k * (1 + 0.134145 * z * z), k * 0.26829 * z
    s = torch.sigmoid(q)
    off = (q.abs() * 1.5 + 24) * 2 * F32 * (s + z.abs() * s * (1 - s) * dq)
    return (s + z * s * (1 - s) * dq, off,
            s * (1 - s) * (2 * dq + z * ddq + z * dq * dq * (1 - 2 * s)))


class Code:
    """Slopes as the forward hands them to the backward: float32 bits shifted right by S, in steps of 1 / 32767."""

    def __init__(self, dtype):
        self.S, one = (1, 31700) if dtype == torch.float16 else (2, 32230)
        self.step = torch.tensor(1.0) / 32767
        self.bias = (self.step * one).view(torch.int32).item() - (0x3F800000 >> self.S)

    def encode(self, s):
        u = s.float().view(torch.int32) & 0x7FFFFFFF
        return torch.copysign(torch.round(((u >> self.S) + self.bias).view(torch.float32) * 32767), s.float())

    def decode(self, c):
        u = (c.abs() * self.step).view(torch.int32)
        return torch.copysign(((u.clamp(min=self.bias) - self.bias) << self.S).view(torch.float32), c).double()

    def __call__(self, s):
        return self.decode(self.encode(s))


def bound(z, name, dtype):
    """(slope, the least and the most of what comes back) in 64 bits."""
    s, off, _ = slope(z, name)
    code = Code(dtype)
    return s, code(s - off), code(s + off)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_code(dtype):
    """Half a step: 2^-15 (bf16 2^-14) from 1/2 to 1, 2^-14 (2^-13) of the slope to 0.283 (0.0708), twice that for each
    two (four) powers of two more; 2^-30 (2^-60) is not zero; values that the code holds are kept. (The
    bits shifted out and 32767 instead of 32768 steps add less than 0.5 % to half a step.)"""
    code = Code(dtype)
    S, edge = code.S, (0.283 if code.S == 1 else 0.0708)
    c = torch.arange(-32766, 32767).float()
    assert torch.equal(code.encode(code.decode(c)), c) and (code.decode(c).diff() > 0).all()
    assert code(torch.tensor([0.0, 1.0])).tolist() == [0.0, 1.0] and code.encode(torch.tensor(1.12903)) < 32766
    s = torch.logspace(math.log10(2.0 ** -30), math.log10(1.129), 400000, dtype=torch.float64)
    off = (code(s) - s.float().double()).abs()
    assert (off[(s >= 0.5) & (s < 1)] <= 2.0 ** (S - 16) * 1.005).all()
    steps = (torch.log2(edge / s) / 2 ** S).ceil().clamp(min=0)
    assert (off <= s * 2.0 ** (steps + S - 15) * 1.005).all()
    assert code(torch.tensor(2.0 ** (-30 if S == 1 else -60))) > 0


@pytest.mark.parametrize("name", SMOOTH)
@pytest.mark.parametrize("dtype", TYPES)
def test_each_slope(name, dtype):
    """One argument a column, a second row whose slope is one: db is slope - c, c near the slope, so that its rounding
    to 16 bits leaves the slope's own digits."""
    z = torch.cat([torch.linspace(-13, 8, 4000), torch.linspace(-1, 1, 1000)]).to(dtype).unique()
    zd = z.double()
    want, least, most = bound(zd, name, dtype)
    c = want.to(dtype)
    w = torch.stack([z, torch.full_like(z, 100.0)], 1).cuda()
    x = torch.eye(2, dtype=dtype, device="cuda")
    b = torch.zeros(len(z), dtype=dtype, device="cuda", requires_grad=True)
    dy = torch.stack([torch.ones_like(z), -c]).cuda()
    (db,) = torch.autograd.grad(fm.linear(x, w, b, name), b, dy)
    got = db.cpu().double() + c.double()
    # the difference in float32, and its rounding to 16 bits
    off = UNIT[dtype] * db.cpu().double().abs() * 1.01 + 2 * F32 * want.abs() + TINY[dtype]
    ok = (got >= least - off) & (got <= most + off)
    at = (~ok).int().argmax()
    assert ok.all(), [t[at].item() for t in (z, got, want, least, most, off)]
    # without a row beside it a slope far out is there by itself
    (db,) = torch.autograd.grad(fm.linear(x[:1], w, b, name), b, torch.ones(1, len(z), dtype=dtype, device="cuda"))
    held = torch.minimum(least.abs(), most.abs()) * (least * most > 0) > 2 * TINY[dtype]
    assert held.sum() > 0.6 * len(z) and (db.cpu()[held] != 0).all()


def test_slopes_of_zero_one_and_nan():
    for dtype in TYPES:
        z = torch.tensor([-60.0, 60.0, float("nan")], dtype=dtype)
        for name in SMOOTH:
            b = torch.zeros(3, dtype=dtype, device="cuda", requires_grad=True)
            y = fm.linear(torch.ones(1, 1, dtype=dtype, device="cuda"), z[:, None].cuda(), b, name)
            (db,) = torch.autograd.grad(y, b, torch.full((1, 3), 3.0, dtype=dtype, device="cuda"))
            assert db[:2].tolist() == [0.0, 3.0] and math.isnan(db[2].item())
        z[2] = 0.5
        b = torch.zeros(3, dtype=dtype, device="cuda", requires_grad=True)
        y = fm.linear(torch.ones(1, 1, dtype=dtype, device="cuda"), z[:, None].cuda(), b, "relu")
        (db,) = torch.autograd.grad(y, b, torch.full((1, 3), 3.0, dtype=dtype, device="cuda"))
        assert db.tolist() == [0.0, 3.0, 3.0]


def problem(M, N, K, dtype, mean, spread, seed, size):
    """Arguments about `mean`, gradients of `size`."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).to(dtype)
    w = (spread * torch.randn(N, K, generator=g) / math.sqrt(K)).to(dtype)
    b = torch.full((N,), mean).to(dtype)
    return x, w, b, (size * torch.randn(M, N, generator=g)).to(dtype)


# arguments where all slopes are small; float16's gradients carry a loss scale, as they do in earnest
@pytest.mark.parametrize("dtype,size", [(torch.float16, 256.0), (torch.bfloat16, 0.02)])
@pytest.mark.parametrize("name,mean", [("gelu", -5.0), ("gelu_tanh", -4.5), ("silu", -13.0), ("gelu", 0.0), ("silu", 0.0),
                                       ("gelu_tanh", 3.0)])
@pytest.mark.parametrize("M,N,K", [(60, 40, 48), (700, 264, 72), (4096, 1032, 128)])
def test_gradients_of_arguments_far_out(M, N, K, name, mean, dtype, size):
    x, w, b, dy = problem(M, N, K, dtype, mean, 0.25 if mean else 1.0, M + N, size)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(fm.linear(*leaves, name), leaves, dy.cuda())
    u, tiny = UNIT[dtype], TINY[dtype]
    xd, wd, bd, dyd = (t.double() for t in (x, w, b, dy))
    z = xd @ wd.t() + bd
    ze = F32 * (K + 4) * (xd.abs() @ wd.abs().t() + bd.abs())
    s, least, most = bound(z, name, dtype)
    se = torch.maximum((most - s).abs(), (least - s).abs())
    _, _, ds = slope(z, name)
    # z's own error moves the slope by its slope there (a second one bounds how that changes over ze)
    dz, dze = dyd * s, dyd.abs() * (se + ze * (1.1 * ds.abs() + 4 * ze))
    dzr = dze + u * (dz.abs() + dze) + tiny
    for got, want, tol in ((dx, dz @ wd, dzr @ wd.abs() + F32 * (N + 4) * (dz.abs() @ wd.abs())),
                           (dw, dz.t() @ xd, dzr.t() @ xd.abs() + F32 * (M + 4) * (dz.abs().t() @ xd.abs())),
                           (db, dz.sum(0), dze.sum(0) + F32 * (M + 4) * dz.abs().sum(0))):
        got, tol = got.cpu().double(), tol + u * want.abs() + tiny
        past = want.abs() + tol >= torch.finfo(dtype).max  # past the type's range, or so near that it rounds out of it
        assert (torch.isinf(got) <= past).all() and (want.abs() - tol < 1.01 * torch.finfo(dtype).max)[~torch.isinf(got)].all()
        got, want, tol = got[~past], want[~past], tol[~past]
        off = (got - want).abs() / tol
        assert off.max() <= 1.01, off.max().item()
        # and by their own size: roundings are not all of one sign
        assert (got - want).norm() <= (0.1 if dtype == torch.float16 else 0.02) * want.norm()


@pytest.mark.parametrize("name", ["gelu", "silu"])
def test_more_than_2_32_slopes(name):
    """Gradients of a few rows of 4.3e9 outputs, the last ones among them."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of free GPU memory")
    dtype, (M, N, K) = torch.float16, ((1 << 20) + 5, 4104, 16)
    g = torch.Generator().manual_seed(5)
    pick = torch.tensor([0, 1, 1023, 1 << 19, 1046527, 1046528, 1 << 20, M - 2, M - 1])  # 1046528 * 4104 passes 2^32
    part = torch.randn(4099, K, generator=g).to(dtype)
    w, b = torch.randn(N, K, generator=g).to(dtype), torch.full((N,), -4.0).to(dtype)
    dyp = (64 * torch.randn(len(pick), N, generator=g)).to(dtype)
    x = part.cuda().repeat(-(-M // 4099), 1)[:M].requires_grad_(True)
    leaves = [x, w.cuda().requires_grad_(True), b.cuda().requires_grad_(True)]
    dy = torch.zeros(M, N, dtype=dtype, device="cuda")
    dy[pick.cuda()] = dyp.cuda()
    dx, dw, db = torch.autograd.grad(fm.linear(*leaves, name), leaves, dy)
    assert not dx[5000].any() and not dx[M - 3].any()
    u, tiny = UNIT[dtype], TINY[dtype]
    xd, wd, bd, dyd = part[pick % 4099].double(), w.double(), b.double(), dyp.double()
    z = xd @ wd.t() + bd
    ze = F32 * (K + 4) * (xd.abs() @ wd.abs().t() + bd.abs())
    s, least, most = bound(z, name, dtype)
    _, _, ds = slope(z, name)
    dz, dze = dyd * s, dyd.abs() * (torch.maximum((most - s).abs(), (least - s).abs()) + ze * (1.1 * ds.abs() + 4 * ze))
    dzr = dze + u * (dz.abs() + dze) + tiny
    for got, want, tol in ((dx[pick.cuda()], dz @ wd, dzr @ wd.abs() + F32 * (N + 4) * (dz.abs() @ wd.abs())),
                           (dw, dz.t() @ xd, dzr.t() @ xd.abs() + F32 * (len(pick) + 4) * (dz.abs().t() @ xd.abs())),
                           (db, dz.sum(0), dze.sum(0) + F32 * (len(pick) + 4) * dz.abs().sum(0))):
        off = (got.cpu().double() - want).abs() / (tol + u * want.abs() + tiny)
        assert off.max() <= 1.01, off.max().item()
