"""Measured cases of the trained layers around MaxSim: linear, layer norm, AdamW.

Each case is one call of a public function of flash_maxsim_amd on data that is
already on the GPU, as a program that trains or serves a token encoder's last
layers calls it: hidden states are normalised and projected to the width that
MaxSim scores, gradients come back from the scores, the optimizer moves the
weights. "train" cases are one forward and one backward pass.

`listed` holds the sizes that stand for each use, `draw` more of the same uses
over their whole range. With `own` false the operators are computed in their
plain form, elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 256  # elements that share a scale in 8-bit optimizer states
BETA1, BETA2, EPS, LR, DECAY, STEP = 0.9, 0.999, 1e-8, 1e-3, 0.01, 10


def listed():
    return [
        # one query's hidden states projected to the scored width: the smallest call, where latency counts
        {"name": "project_query", "op": "linear", "dtype": "bf16", "M": 32, "K": 768, "N": 128, "act": "none",
         "residual": False, "train": False},
        # documents at indexing time, first layer of a feed-forward pair
        {"name": "feed_forward_up", "op": "linear", "dtype": "bf16", "M": 8192, "K": 1024, "N": 4096, "act": "gelu",
         "residual": False, "train": False},
        # its second layer, back onto the hidden states; a ragged batch's odd token count
        {"name": "feed_forward_down", "op": "linear", "dtype": "f16", "M": 7777, "K": 4096, "N": 1024, "act": "none",
         "residual": True, "train": False},
        # training step of the projection over a batch of documents, wide hidden states
        {"name": "train_project", "op": "linear", "dtype": "bf16", "M": 24576, "K": 2048, "N": 128, "act": "none",
         "residual": False, "train": True},
        # training step of a feed-forward layer: the largest product
        {"name": "train_feed_forward", "op": "linear", "dtype": "bf16", "M": 16384, "K": 1024, "N": 4096,
         "act": "gelu", "residual": False, "train": True},
        # an adapter of odd widths, every size off the tiles
        {"name": "train_odd", "op": "linear", "dtype": "f16", "M": 1003, "K": 300, "N": 77, "act": "silu",
         "residual": True, "train": True},
        # one query's hidden states normalised
        {"name": "norm_query", "op": "norm", "dtype": "bf16", "M": 32, "d": 768, "train": False},
        # training step over a batch of documents
        {"name": "train_norm", "op": "norm", "dtype": "bf16", "M": 65536, "d": 1024, "train": True},
        # float32 hidden states of an odd width
        {"name": "train_norm_odd", "op": "norm", "dtype": "f32", "M": 1537, "d": 771, "train": True},
        # the head alone is trained: a handful of small tensors
        {"name": "adamw_head", "op": "adamw", "dtype": "f32", "bits": 32, "tensors": 6, "total": 200_000,
         "copies": False},
        # the whole encoder in float32 with bf16 copies for the next forward pass, many tensors
        {"name": "adamw_encoder", "op": "adamw", "dtype": "f32", "bits": 32, "tensors": 150, "total": 64_000_000,
         "copies": True},
        # the same with 8-bit states, parameters kept in bf16 alone
        {"name": "adamw_8bit", "op": "adamw", "dtype": "bf16", "bits": 8, "tensors": 150, "total": 64_000_000,
         "copies": False},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "adamw"])
    if op == "linear":
        K = rng.choice([128, 256, 384, 768, 1024, 2048, 4096, _spread(rng, 16, 4096)])
        N = rng.choice([128, 128, 96, 768, 1024, 4096, _spread(rng, 16, 4096)])
        train = rng.random() < 0.5
        M = _spread(rng, 1, max(2, min(65536, int(2 ** 36 / (K * N) / (1 if train else 2)))))
        return {"op": "linear", "dtype": rng.choice(["bf16", "f16"]), "M": M, "K": K, "N": N,
                "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "residual": rng.random() < 0.4,
                "train": train}
    if op == "norm":
        d = rng.choice([128, 256, 768, 1024, 2048, _spread(rng, 16, 8192)])
        return {"op": "norm", "dtype": rng.choice(["bf16", "f16", "f32"]), "M": _spread(rng, 1, min(65536, 2 ** 25 // d)),
                "d": d, "train": rng.random() < 0.6}
    bits = rng.choice([32, 8])
    dtype = rng.choice(["f32", "bf16", "f16"])
    total = _spread(rng, 10_000, 32_000_000)
    return {"op": "adamw", "dtype": dtype, "bits": bits, "tensors": rng.randint(1, 150), "total": total,
            "copies": dtype == "f32" and rng.random() < 0.5}


# ---- inputs ----

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _hidden(g, M, d):
    """Hidden states: unit variance about a mean of their own per row, a few wide channels, as encoders have them."""
    x = _randn(g, M, d)
    x *= 1.0 + 4.0 * (torch.rand(d, generator=g, device=DEV) < 0.01)
    return x.add_(0.3 * _randn(g, M, 1))


def _sizes(case):
    """Element counts of the tensors: vectors (biases, norms) between matrices of uneven sizes that make up the total."""
    n, total = case["tensors"], case["total"]
    weights = [1.0 if i % 3 == 0 else 0.002 if i % 3 == 1 else 2.5 for i in range(n)]
    return [max(1, int(total * w / sum(weights)) - (i % 5)) for i, w in enumerate(weights)]


def _encode(m, signed):
    """8-bit codes of rows of BLOCK values and the scale of each row (see _decode)."""
    top = 127 if signed else 255
    big = m.abs().amax(1, keepdim=True)
    whole = torch.full_like(big, float(top * top))
    tiny = big < 2.0 ** -110  # held as zeros
    inv = torch.where(tiny, torch.zeros_like(big), whole / torch.where(tiny, torch.ones_like(big), big))
    y = m.abs() * inv
    c = torch.round(torch.sqrt(y))  # the nearest code, settled by comparisons that are exact in 32 bits
    c = c + (y >= c * c + c + 0.25)
    c = c - (y < c * c - c + 0.25).to(c.dtype) * (c > 0)
    c = c.clamp(max=top)
    if signed:
        c = torch.where(m < 0, -c, c).to(torch.int8)
    else:
        c = torch.where((m > 0) & ~tiny, c.clamp(min=1), c).to(torch.uint8)
    return c, torch.where(tiny, torch.zeros_like(big), big) / whole


def _decode(c, scale):
    """The values of 8-bit codes: c |c| times the row's scale."""
    f = c.to(torch.float32)
    return (f * f.abs()) * scale


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "linear":
        M, K, N, dt = case["M"], case["K"], case["N"], DTYPES[case["dtype"]]
        s = {"x": _hidden(g, M, K).to(dt), "w": (_randn(g, N, K) / math.sqrt(K)).to(dt), "b": (0.1 * _randn(g, N)).to(dt),
             "r": _hidden(g, M, N).to(dt) if case["residual"] else None}
        if case["train"]:
            s["dy"] = (_randn(g, M, N) * 0.02).to(dt)
    elif case["op"] == "norm":
        M, d, dt = case["M"], case["d"], DTYPES[case["dtype"]]
        s = {"x": _hidden(g, M, d).to(dt), "w": (1.0 + 0.1 * _randn(g, d)).to(dt), "b": (0.1 * _randn(g, d)).to(dt)}
        if case["train"]:
            s["dy"] = (_randn(g, M, d) * 0.02).to(dt)
    else:
        sizes = _sizes(case)
        starts, total = [], 0
        for n in sizes:  # every tensor begins at a block of its own in the flat buffers
            starts.append(total)
            total += -(-n // BLOCK) * BLOCK
        live = torch.zeros(total, dtype=torch.bool, device=DEV)
        for a, n in zip(starts, sizes):
            live[a:a + n] = True
        spread = torch.exp(1.5 * _randn(g, total))  # gradients differ in size from weight to weight
        flat = {"p": (0.03 * _randn(g, total) * live).to(DTYPES[case["dtype"]]),
                "g": (1e-3 * _randn(g, total) * spread * live).to(DTYPES[case["dtype"]])}
        m, v = 2e-4 * _randn(g, total) * spread * live, (3e-4 * spread * live) ** 2
        s = {"flat": flat, "step": STEP, "scale": torch.full((), 0.8, device=DEV)}
        if case["bits"] == 8:
            flat["m"], ms = _encode(m.view(-1, BLOCK), True)
            flat["v"], vs = _encode(torch.sqrt(v).view(-1, BLOCK), False)
            flat["m"], flat["v"], flat["ms"], flat["vs"] = flat["m"].view(-1), flat["v"].view(-1), ms.view(-1), vs.view(-1)
        else:
            flat["m"], flat["v"] = m, v
        if case["copies"]:
            flat["c"] = flat["p"].to(torch.bfloat16)
        part = {k: [t[a // BLOCK:-(-(a + n) // BLOCK)] if k in ("ms", "vs") else t[a:a + n] for a, n in zip(starts, sizes)]
                for k, t in flat.items()}
        if case["bits"] == 8:  # a moment: its codes and their scales
            part["m"], part["v"] = list(zip(part["m"], part["ms"])), list(zip(part["v"], part["vs"]))
        s["tensors"] = part
    s["case"] = dict(case)
    return s


# ---- the plain forms; with dtype float64 the definition in 64 bits is written apart, below ----

def _act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_grad(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * k * (1.0 + 0.134145 * z * z)
    if name == "silu":
        e = 1.0 / (1.0 + torch.exp(-z))
        return e * (1.0 + z * (1.0 - e))
    return torch.ones_like(z)


def _plain_linear(s, c):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t() + s["b"].float()
    y = _act(z, c["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    out = {"y": y.to(dt)}
    if c["train"]:
        dz = s["dy"].float()
        if c["act"] != "none":
            dz = dz * _act_grad(z, c["act"])
        out |= {"dx": (dz @ w).to(dt), "dw": (dz.t() @ x).to(dt), "db": dz.sum(0).to(dt)}
        if s["r"] is not None:
            out["dr"] = s["dy"]
    return out


def _plain_norm(s, c):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    x = x - x.mean(1, keepdim=True)
    rs = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-5)
    xh = x * rs
    out = {"y": (xh * w + s["b"].float()).to(dt)}
    if c["train"]:
        dy = s["dy"].float()
        wdy = dy * w
        dx = rs * (wdy - wdy.mean(1, keepdim=True) - xh * (wdy * xh).mean(1, keepdim=True))
        out |= {"dx": dx.to(dt), "dw": (dy * xh).sum(0).to(dt), "db": dy.sum(0).to(dt)}
    return out


def _plain_adamw(s, c):
    f, t = s["flat"], s["step"]
    p, g = f["p"].float(), f["g"].float() * s["scale"]
    if c["bits"] == 8:
        m = _decode(f["m"].view(-1, BLOCK), f["ms"].view(-1, 1)).view(-1)
        r = _decode(f["v"].view(-1, BLOCK), f["vs"].view(-1, 1)).view(-1)
        v = r * r
    else:
        m, v = f["m"], f["v"]
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    r = torch.sqrt(v)
    p = p * (1.0 - LR * DECAY) - (m / (r * (1.0 / math.sqrt(1.0 - BETA2 ** t)) + EPS)) * (LR / (1.0 - BETA1 ** t))
    f["p"].copy_(p)
    if c["copies"]:
        f["c"].copy_(p)
    if c["bits"] == 8:
        cm, ms = _encode(m.view(-1, BLOCK), True)
        cv, vs = _encode(r.view(-1, BLOCK), False)
        f["m"].copy_(cm.view(-1)), f["ms"].copy_(ms.view(-1)), f["v"].copy_(cv.view(-1)), f["vs"].copy_(vs.view(-1))
        r = _decode(cv, vs)
        return {"p": f["p"], "m": _decode(cm, ms).view(-1), "v": (r * r).view(-1)}
    f["m"].copy_(m), f["v"].copy_(v)
    return {k: f[k] for k in ("p", "m", "v", "c") if k in f}


# ---- the framework's operators ----

def _own_linear(s, c):
    import flash_maxsim_amd as fm

    act = None if c["act"] == "none" else c["act"]
    if not c["train"]:
        return {"y": fm.linear(s["x"], s["w"], s["b"], act, s["r"])}
    leaves = [s[k].requires_grad_(True) for k in ("x", "w", "b", "r") if s[k] is not None]
    y = fm.linear(s["x"], s["w"], s["b"], act, s["r"])
    return {"y": y} | dict(zip(("dx", "dw", "db", "dr"), torch.autograd.grad(y, leaves, s["dy"])))


def _own_norm(s, c):
    import flash_maxsim_amd as fm

    if not c["train"]:
        return {"y": fm.layer_norm(s["x"], s["w"], s["b"], eps=1e-5)}
    leaves = [s[k].requires_grad_(True) for k in ("x", "w", "b")]
    y = fm.layer_norm(s["x"], s["w"], s["b"], eps=1e-5)
    return {"y": y} | dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, s["dy"])))


def _own_adamw(s, c):
    import flash_maxsim_amd as fm

    f, t = s["flat"], s["tensors"]
    fm.adamw_step(t["p"], t["g"], t["m"], t["v"], s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                  grad_scale=s["scale"], copies=t.get("c"))
    if c["bits"] == 8:
        return {"p": f["p"], "m": fm.dequantize_adamw((f["m"], f["ms"])), "v": fm.dequantize_adamw((f["v"], f["vs"]))}
    return {k: f[k] for k in ("p", "m", "v", "c") if k in f}


def run(state):
    c = state["case"]
    if own:
        return {"linear": _own_linear, "norm": _own_norm, "adamw": _own_adamw}[c["op"]](state, c)
    return {"linear": _plain_linear, "norm": _plain_norm, "adamw": _plain_adamw}[c["op"]](state, c)


def work(case):
    if case["op"] == "linear":
        M, K, N, r = case["M"], case["K"], case["N"], 1 if case["residual"] else 0
        values = M * K + N * K + N + M * N * (1 + r)
        flops = 2 * M * K * N
        if case["train"]:  # x, w and z (or nothing of it) are read once for both passes
            values += M * N + M * K + N * K + N
            flops *= 3
        return {"bytes": 2 * values, "flops": flops}
    if case["op"] == "norm":
        M, d, size = case["M"], case["d"], 4 if case["dtype"] == "f32" else 2
        values = 2 * M * d + 2 * d
        if case["train"]:
            values += 2 * M * d + 2 * d
        return {"bytes": size * values, "flops": (20 if case["train"] else 8) * M * d}
    n = sum(_sizes(case))
    size = 4 if case["dtype"] == "f32" else 2
    per = 3 * size + (2 if case["copies"] else 0)
    if case["bits"] == 32:
        return {"bytes": n * (per + 16), "flops": 16 * n}
    scales = 2 * 4 * (n // BLOCK + case["tensors"])
    # the states are read, written, and returned as the values that they stand for
    return {"bytes": n * (per + 4 + 8) + 2 * scales, "flops": 40 * n}


# ---- the definitions in 64 bits ----

def _exact_linear(s, c):
    x, w, b = (s[k].double() for k in ("x", "w", "b"))
    z = torch.addmm(b, x, w.t()).requires_grad_(c["train"])
    a = {"none": lambda q: q, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda q: torch.nn.functional.gelu(q, approximate="tanh")}[c["act"]](z)
    out = {"y": (a if s["r"] is None else a + s["r"].double()).detach()}
    if c["train"]:
        dz = torch.autograd.grad(a, z, s["dy"].double())[0] if c["act"] != "none" else s["dy"].double()
        out |= {"dx": torch.mm(dz, w), "dw": torch.mm(dz.t().contiguous(), x), "db": dz.sum(0)}
        if s["r"] is not None:
            out["dr"] = s["dy"].double()
    return out


def _exact_norm(s, c):
    x, w, b = (s[k].double().requires_grad_(c["train"]) for k in ("x", "w", "b"))
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    y = torch.addcmul(b, (x - mean) * torch.rsqrt(var + 1e-5), w)
    out = {"y": y.detach()}
    if c["train"]:
        out |= dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), s["dy"].double())))
    return out


def _exact_code(x, top, least):
    """The values that top^2 levels c^2 / top^2 of each row's largest stand for, the nearest root of each value taken."""
    big = x.abs().amax(1, keepdim=True)
    big = torch.where(big > 0, big, torch.ones_like(big))
    c = torch.round(torch.sqrt(x.abs() / big) * top).clamp(max=top)
    c = torch.where(x != 0, c.clamp(min=least), c)
    return torch.sign(x) * (c / top) ** 2 * big


def _exact_adamw(s, c):
    f, t = s["flat"], s["step"]
    p, g, m, v = (f[k].double() for k in ("p", "g", "m", "v"))
    g = g * float(s["scale"])
    if c["bits"] == 8:
        m = (m * m.abs()).view(-1, BLOCK).mul(f["ms"].double().view(-1, 1)).view(-1)
        v = (v * v).view(-1, BLOCK).mul(f["vs"].double().view(-1, 1)).view(-1).square()
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g * g, v, BETA2)
    p = p - LR * DECAY * p
    p = p - LR * (m / (1.0 - BETA1 ** t)) / (torch.sqrt(v / (1.0 - BETA2 ** t)) + EPS)
    out = {"p": p, "m": m, "v": v}
    if c["bits"] == 8:
        out["m"] = _exact_code(m.view(-1, BLOCK), 127, 0).view(-1)
        out["v"] = _exact_code(torch.sqrt(v).view(-1, BLOCK), 255, 1).view(-1).square()
    if c["copies"]:
        out["c"] = p
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"linear": _exact_linear, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](s, s["case"])
