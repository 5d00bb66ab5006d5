"""Measured cases of the encoder block around MaxSim: gated feed-forward, residual norm, embedding, Muon.

Each case is one call of a public function of flash_maxsim_amd on data that is
already on the GPU, as a program that trains or serves a token encoder calls it:
token ids are looked up, the block's gated feed-forward layer runs, its output is
normalised, gated and added to the hidden states, which are normalised for the
next block, gradients come back through all of that, and the optimizer moves the
weight matrices by orthogonalised updates. "train" cases are one forward and one
backward pass.

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
EPS = 1e-5
# the optimizer's constants: learning rate, momentum, decay, the steps of the iteration and its polynomial
LR, MU, DECAY, STEPS, POLY = 0.02, 0.95, 0.01, 5, (3.4445, -4.7750, 2.0315)


def listed():
    return [
        # one query's tokens through a block's gated layer: the smallest call, where latency counts
        {"name": "gate_query", "op": "gated", "dtype": "bf16", "M": 32, "K": 768, "N": 1152, "act": "gelu", "bias": False,
         "train": False},
        # documents at indexing time
        {"name": "gate_index", "op": "gated", "dtype": "bf16", "M": 8192, "K": 1024, "N": 4096, "act": "silu", "bias": False,
         "train": False},
        # training step of the layer over a batch of documents: the largest products
        {"name": "train_gate", "op": "gated", "dtype": "bf16", "M": 16384, "K": 1024, "N": 2816, "act": "silu",
         "bias": False, "train": True},
        # an adapter of odd widths with biases, every size off the tiles
        {"name": "train_gate_odd", "op": "gated", "dtype": "f16", "M": 1003, "K": 300, "N": 77, "act": "gelu_tanh",
         "bias": True, "train": True},
        # one query between two blocks: add and normalise
        {"name": "stream_query", "op": "stream", "dtype": "bf16", "M": 32, "d": 768, "norm": "layer", "post": False,
         "gate": False, "scale": False, "alpha": 1.0, "train": False},
        # training step over a batch of documents: block output normalised, gated and scaled onto the hidden states
        {"name": "train_stream", "op": "stream", "dtype": "bf16", "M": 65536, "d": 1024, "norm": "rms", "post": True,
         "gate": True, "scale": True, "alpha": 1.0, "train": True},
        # a ragged batch of an odd width, hidden states scaled up beside the block's output
        {"name": "train_stream_odd", "op": "stream", "dtype": "f16", "M": 1537, "d": 771, "norm": "layer", "post": True,
         "gate": False, "scale": True, "alpha": 1.5, "train": True},
        # one query's ids looked up
        {"name": "embed_query", "op": "embed", "dtype": "bf16", "T": 32, "V": 32768, "d": 768, "train": False},
        # training step of the table over a batch of documents: few ids make up most of the tokens, most ids are absent
        {"name": "train_embed", "op": "embed", "dtype": "bf16", "T": 65536, "V": 131072, "d": 1024, "train": True},
        # a small float32 table of an odd width
        {"name": "train_embed_odd", "op": "embed", "dtype": "f32", "T": 5001, "V": 1009, "d": 300, "train": True},
        # the matrices of a small head, orthogonalised
        {"name": "muon_head", "op": "muon", "form": "update", "dtype": "bf16", "layers": 1, "h": 256, "f": 1024, "out": 128},
        # the optimizer's step over the feed-forward matrices of a whole encoder
        {"name": "muon_encoder", "op": "muon", "form": "step", "dtype": "bf16", "layers": 8, "h": 1024, "f": 4096, "out": 128},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gated", "gated", "stream", "embed", "muon"])
    if op == "gated":
        K = rng.choice([128, 256, 384, 768, 1024, 2048, _spread(rng, 16, 2048)])
        N = rng.choice([256, 512, 1024, 1152, 2816, 4096, _spread(rng, 16, 4096)])
        train = rng.random() < 0.5
        M = _spread(rng, 1, max(2, min(32768, int(2 ** 35 / (K * N) / (1 if train else 2)))))
        return {"op": "gated", "dtype": rng.choice(["bf16", "f16"]), "M": M, "K": K, "N": N,
                "act": rng.choice(["silu", "gelu", "gelu_tanh", "relu"]), "bias": rng.random() < 0.3, "train": train}
    if op == "stream":
        d = rng.choice([128, 256, 768, 1024, 2048, _spread(rng, 16, 4096)])
        post = rng.random() < 0.5
        return {"op": "stream", "dtype": rng.choice(["bf16", "f16"]), "M": _spread(rng, 1, min(65536, 2 ** 25 // d)), "d": d,
                "norm": rng.choice(["layer", "rms"]), "post": post, "gate": rng.random() < 0.4, "scale": rng.random() < 0.5,
                "alpha": rng.choice([1.0, 1.0, 2.0]), "train": rng.random() < 0.6}
    if op == "embed":
        d = rng.choice([128, 256, 768, 1024, _spread(rng, 16, 2048)])
        V = _spread(rng, 100, min(131072, 2 ** 26 // d))
        return {"op": "embed", "dtype": rng.choice(["bf16", "f16", "f32"]), "T": _spread(rng, 1, min(65536, 2 ** 25 // d)),
                "V": V, "d": d, "train": rng.random() < 0.7}
    h = rng.choice([128, 256, 384, 512, _spread(rng, 24, 1024), _spread(rng, 24, 1024)])
    f = rng.choice([2 * h, 4 * h, _spread(rng, h, 4 * h)])
    return {"op": "muon", "form": rng.choice(["update", "step"]), "dtype": "bf16",
            "layers": rng.randint(1, max(1, min(8, 2 ** 30 // (h * h * f)))), "h": h, "f": f,
            "out": rng.choice([96, 128, _spread(rng, 16, 256), _spread(rng, 16, 256)])}


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


def _matrices(case):
    """(count, rows, columns) of the weight matrices: gate and up, down, and the projection to the scored width."""
    layers, h, f, out = case["layers"], case["h"], case["f"], case["out"]
    return [(2 * layers, f, h), (layers, h, f), (1, out, h)]


def _update(g, count, rows, cols):
    """Gradients of matrices: a few directions that the batch agrees on, falling off, over a floor of noise."""
    r = min(32, rows, cols)
    fall = torch.arange(1, r + 1, device=DEV, dtype=torch.float32) ** -0.7
    x = torch.bmm(_randn(g, count, rows, r) * fall, _randn(g, count, r, cols))
    return x.add_(_randn(g, count, rows, cols) * 0.5).mul_(1e-3)


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "gated":
        M, K, N = case["M"], case["K"], case["N"]
        s = {"x": _hidden(g, M, K).to(dt), "wg": (_randn(g, N, K) / math.sqrt(K)).to(dt),
             "wu": (_randn(g, N, K) / math.sqrt(K)).to(dt)}
        s["bg"], s["bu"] = ((0.1 * _randn(g, N)).to(dt), (0.1 * _randn(g, N)).to(dt)) if case["bias"] else (None, None)
        if case["train"]:
            s["dy"] = (_randn(g, M, N) * 0.02).to(dt)
    elif case["op"] == "stream":
        M, d = case["M"], case["d"]
        bias = case["norm"] == "layer"
        s = {"x": (0.5 * _hidden(g, M, d)).to(dt), "r": _hidden(g, M, d).to(dt), "w": (1.0 + 0.1 * _randn(g, d)).to(dt),
             "b": (0.1 * _randn(g, d)).to(dt) if bias else None,
             "pw": (1.0 + 0.1 * _randn(g, d)).to(dt) if case["post"] else None,
             "pb": (0.1 * _randn(g, d)).to(dt) if case["post"] and bias else None,
             "gate": torch.sigmoid(_randn(g, M, d)).to(dt) if case["gate"] else None,
             "scale": (0.5 + 0.1 * _randn(g, d)).to(dt) if case["scale"] else None}
        if case["train"]:  # gradients of both results: the hidden states go on, and the next block's input comes of them
            s["dh"], s["dy"] = (_randn(g, M, d) * 0.02).to(dt), (_randn(g, M, d) * 0.02).to(dt)
    elif case["op"] == "embed":
        T, V, d = case["T"], case["V"], case["d"]
        rank = torch.exp(torch.rand(T, generator=g, device=DEV) * math.log(V)).long() - 1  # frequencies like 1 / rank
        order = torch.randperm(V, generator=g, device=DEV)  # frequent ids lie anywhere in the table
        s = {"ids": order[rank.clamp(0, V - 1)], "w": _randn(g, V, d).mul_(0.02).to(dt)}
        if case["train"]:
            s["dy"] = (_randn(g, T, d) * 0.02).to(dt)
    else:
        shapes = _matrices(case)
        s = {"g": [_update(g, *shape).to(dt) for shape in shapes]}
        if case["form"] == "step":
            s["p"] = [(_randn(g, *shape) * 0.03).to(dt) for shape in shapes]
            s["m"] = [_update(g, *shape) for shape in shapes]
        # the tensors of a program's parameter list, matrices of one shape side by side in memory
        s["lists"] = {k: [t for stack in s[k] for t in stack.unbind(0)] for k in ("g", "p", "m") if k in s}
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
    return z / (1.0 + torch.exp(-z))


def _act_grad(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * k * (1.0 + 0.134145 * z * z)
    e = 1.0 / (1.0 + torch.exp(-z))
    return e * (1.0 + z * (1.0 - e))


def _plain_gated(s, c):
    dt = s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    if c["bias"]:
        g, u = g + s["bg"].float(), u + s["bu"].float()
    a = _act(g, c["act"])
    out = {"y": (a * u).to(dt)}
    if c["train"]:
        dy = s["dy"].float()
        dg, du = dy * u * _act_grad(g, c["act"]), dy * a
        out |= {"dx": (dg @ wg + du @ wu).to(dt), "dwg": (dg.t() @ x).to(dt), "dwu": (du.t() @ x).to(dt)}
        if c["bias"]:
            out |= {"dbg": dg.sum(0).to(dt), "dbu": du.sum(0).to(dt)}
    return out


def _plain_norm(x, kind):
    """x normalised, and the factor of each row."""
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    rs = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    return x * rs, rs


def _plain_norm_grad(dxh, xh, rs, kind):
    dx = dxh - xh * (dxh * xh).mean(1, keepdim=True)
    if kind == "layer":
        dx = dx - dxh.mean(1, keepdim=True)
    return rs * dx


def _plain_stream(s, c):
    dt, kind = s["x"].dtype, c["norm"]
    t = s["x"].float()
    if c["post"]:
        xh, rx = _plain_norm(t, kind)
        t = xh * s["pw"].float()
        if s["pb"] is not None:
            t = t + s["pb"].float()
    k = torch.ones((), device=DEV)
    if c["scale"]:
        k = k * s["scale"].float()
    if c["gate"]:
        k = k * s["gate"].float()
    h = c["alpha"] * s["r"].float() + k * t
    hh, rh = _plain_norm(h, kind)
    y = hh * s["w"].float()
    if s["b"] is not None:
        y = y + s["b"].float()
    out = {"h": h.to(dt), "y": y.to(dt)}
    if c["train"]:
        dy = s["dy"].float()
        dh = s["dh"].float() + _plain_norm_grad(dy * s["w"].float(), hh, rh, kind)
        out |= {"dr": (c["alpha"] * dh).to(dt), "dw": (dy * hh).sum(0).to(dt)}
        if s["b"] is not None:
            out["db"] = dy.sum(0).to(dt)
        if c["scale"]:
            out["dscale"] = (dh * t * s["gate"].float() if c["gate"] else dh * t).sum(0).to(dt)
        if c["gate"]:
            out["dgate"] = (dh * t * s["scale"].float() if c["scale"] else dh * t).to(dt)
        dt_ = dh * k
        if c["post"]:
            out["dpw"] = (dt_ * xh).sum(0).to(dt)
            if s["pb"] is not None:
                out["dpb"] = dt_.sum(0).to(dt)
            dt_ = _plain_norm_grad(dt_ * s["pw"].float(), xh, rx, kind)
        out["dx"] = dt_.to(dt)
    return out


def _plain_embed(s, c):
    dt, k = s["w"].dtype, math.sqrt(c["d"])
    out = {"y": (s["w"][s["ids"]].float() * k).to(dt)}
    if c["train"]:
        dw = torch.zeros(c["V"], c["d"], device=DEV)
        dw.index_add_(0, s["ids"], s["dy"].float() * k)
        out["dw"] = dw.to(dt)
    return out


def _plain_orthogonal(u):
    """The iteration on matrices [count, rows, columns] in 32 bits, the shorter side first."""
    a, b, c = POLY
    tall = u.size(1) > u.size(2)
    x = u.transpose(1, 2).contiguous() if tall else u
    x = x / torch.sqrt((x * x).sum((1, 2), keepdim=True)).clamp(min=1e-7)
    for _ in range(STEPS):
        A = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * A + c * torch.bmm(A, A), x)
    return x.transpose(1, 2) if tall else x


def _plain_muon(s, c):
    out = []
    for i, g in enumerate(s["g"]):
        u = g.float()
        if c["form"] == "update":
            out.append(_plain_orthogonal(u).to(g.dtype))
            continue
        p, m = s["p"][i], s["m"][i]
        m.copy_(MU * m + (1.0 - MU) * u)
        u = _plain_orthogonal((1.0 - MU) * u + MU * m)
        rate = LR * math.sqrt(max(1.0, g.size(1) / g.size(2)))
        p.copy_((p.float() * (1.0 - LR * DECAY) - rate * u).to(p.dtype))
    if c["form"] == "update":
        return {"o": [t for stack in out for t in stack.unbind(0)]}
    return {"p": s["p"], "m": s["m"]}


# ---- the framework's operators ----

def _own_gated(s, c):
    import flash_maxsim_amd as fm

    args = s["x"], s["wg"], s["wu"], s["bg"], s["bu"], c["act"]
    if not c["train"]:
        return {"y": fm.gated_linear(*args)}
    names = [k for k in ("x", "wg", "wu", "bg", "bu") if s[k] is not None]
    leaves = [s[k].requires_grad_(True) for k in names]
    y = fm.gated_linear(*args)
    return {"y": y} | dict(zip(("d" + k for k in names), torch.autograd.grad(y, leaves, s["dy"])))


def _own_stream(s, c):
    import flash_maxsim_amd as fm

    names = [k for k in ("x", "r", "w", "b", "pw", "pb", "gate", "scale") if s[k] is not None]
    leaves = [s[k].requires_grad_(True) for k in names] if c["train"] else []
    h, y = fm.residual_norm(s["x"], s["r"], s["w"], s["b"], norm=c["norm"], eps=EPS, post_norm=c["post"], post_weight=s["pw"],
                            post_bias=s["pb"], gate=s["gate"], scale=s["scale"], residual_scale=c["alpha"])
    out = {"h": h, "y": y}
    if c["train"]:
        out |= dict(zip(("d" + k for k in names), torch.autograd.grad((h, y), leaves, (s["dh"], s["dy"]))))
    return out


def _own_embed(s, c):
    import flash_maxsim_amd as fm

    if not c["train"]:
        return {"y": fm.embedding(s["ids"], s["w"], scale=math.sqrt(c["d"]))}
    w = s["w"].requires_grad_(True)
    y = fm.embedding(s["ids"], w, scale=math.sqrt(c["d"]))
    return {"y": y, "dw": torch.autograd.grad(y, w, s["dy"])[0]}


def _own_muon(s, c):
    import flash_maxsim_amd as fm

    t = s["lists"]
    if c["form"] == "update":
        return {"o": fm.orthogonalize(t["g"], steps=STEPS, coefficients=POLY)}
    fm.muon_step(t["p"], t["g"], t["m"], lr=LR, momentum=MU, weight_decay=DECAY, steps=STEPS, coefficients=POLY)
    return {"p": s["p"], "m": s["m"]}


def run(state):
    c = state["case"]
    if own:
        return {"gated": _own_gated, "stream": _own_stream, "embed": _own_embed, "muon": _own_muon}[c["op"]](state, c)
    return {"gated": _plain_gated, "stream": _plain_stream, "embed": _plain_embed, "muon": _plain_muon}[c["op"]](state, c)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "gated":
        M, K, N = case["M"], case["K"], case["N"]
        values = M * K + 2 * N * K + M * N + (2 * N if case["bias"] else 0)
        if case["train"]:  # x and the weights are read once for both passes
            values += M * N + M * K + 2 * N * K + (2 * N if case["bias"] else 0)
        return {"bytes": size * values, "flops": (12 if case["train"] else 4) * M * K * N}
    if case["op"] == "stream":
        M, d = case["M"], case["d"]
        gate, flags = int(case["gate"]), int(case["post"]) + int(case["scale"]) + 1
        values = (4 + gate) * M * d + flags * d
        if case["train"]:
            values += (4 + gate) * M * d + flags * d
        return {"bytes": size * values, "flops": (40 if case["train"] else 14) * M * d}
    if case["op"] == "embed":
        T, V, d = case["T"], case["V"], case["d"]
        values = 2 * T * d + (T * d + V * d if case["train"] else 0)
        return {"bytes": size * values + 8 * T, "flops": (2 if case["train"] else 1) * T * d}
    values = flops = 0
    for count, rows, cols in _matrices(case):
        n, m = min(rows, cols), max(rows, cols)
        values += count * rows * cols
        flops += count * STEPS * (3 * n * n * m + n ** 3)  # of the symmetric products one half
    return {"bytes": values * (2 * size if case["form"] == "update" else 3 * size + 8), "flops": flops}


# ---- the definitions in 64 bits ----

_ACTS = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda q: torch.nn.functional.gelu(q, approximate="tanh")}


def _exact_gated(s, c):
    names = [k for k in ("x", "wg", "wu", "bg", "bu") if s[k] is not None]
    q = {k: s[k].double() for k in names}
    z = torch.mm(q["x"], torch.cat([q["wg"], q["wu"]]).t().contiguous())
    if c["bias"]:
        z = z + torch.cat([q["bg"], q["bu"]])
    z.requires_grad_(c["train"])
    g, u = z.split(c["N"], 1)
    y = _ACTS[c["act"]](g) * u
    out = {"y": y.detach()}
    if c["train"]:
        dg, du = torch.autograd.grad(y, z, s["dy"].double())[0].split(c["N"], 1)
        out |= {"dx": torch.addmm(torch.mm(dg, q["wg"]), du, q["wu"]), "dwg": torch.mm(dg.t().contiguous(), q["x"]),
                "dwu": torch.mm(du.t().contiguous(), q["x"])}
        if c["bias"]:
            out |= {"dbg": dg.sum(0), "dbu": du.sum(0)}
    return out


def _exact_stream(s, c):
    names = [k for k in ("x", "r", "w", "b", "pw", "pb", "gate", "scale") if s[k] is not None]
    q = {k: s[k].double().requires_grad_(c["train"]) for k in names}

    def normal(x, w, b):
        if c["norm"] == "layer":
            var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
            x = (x - mean) * torch.rsqrt(var + EPS)
        else:
            x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
        x = x * q[w]
        return x + q[b] if b in q else x

    t = normal(q["x"], "pw", "pb") if c["post"] else q["x"]
    for k in ("scale", "gate"):
        t = t * q[k] if k in q else t
    h = q["r"] * c["alpha"] + t
    y = normal(h, "w", "b")
    out = {"h": h.detach(), "y": y.detach()}
    if c["train"]:
        out |= dict(zip(("d" + k for k in names),
                        torch.autograd.grad((h, y), [q[k] for k in names], (s["dh"].double(), s["dy"].double()))))
    return out


def _exact_embed(s, c):
    k = math.sqrt(c["d"])
    out = {"y": s["w"].double().index_select(0, s["ids"]) * k}
    if c["train"]:
        dw = torch.zeros(c["V"], c["d"], dtype=torch.float64, device=DEV)
        out["dw"] = dw.index_put_((s["ids"],), s["dy"].double(), accumulate=True).mul_(k)
    return out


def _exact_orthogonal(u):
    """Odd polynomials of the matrices x: p(x) = a x + (b x x^T + c (x x^T)^2) x, each on the last one's result."""
    a, b, c = POLY
    x = u.mT.contiguous() if u.size(1) > u.size(2) else u
    x = x / torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True).clamp(min=1e-7)
    for _ in range(STEPS):
        gram = torch.bmm(x, x.mT.contiguous())
        x = torch.baddbmm(x, torch.baddbmm(gram, gram, gram, beta=b, alpha=c), x, beta=a)
    return x.mT if u.size(1) > u.size(2) else x


def _exact_muon(s, c):
    if c["form"] == "update":
        return {"o": [t for g in s["g"] for t in _exact_orthogonal(g.double()).unbind(0)]}
    out = {"p": [], "m": []}
    for g, p, m in zip(s["g"], s["p"], s["m"]):
        m = torch.lerp(g.double(), m.double(), MU)
        o = _exact_orthogonal(torch.lerp(g.double(), m, MU))
        out["m"].append(m)
        out["p"].append(p.double() * (1.0 - LR * DECAY) - LR * math.sqrt(max(1.0, g.size(1) / g.size(2))) * o)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"gated": _exact_gated, "stream": _exact_stream, "embed": _exact_embed, "muon": _exact_muon}[case["op"]](s, s["case"])
