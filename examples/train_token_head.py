"""Trains the layers between an encoder and MaxSim on synthetic hidden states.

A head turns hidden states into the token embeddings that MaxSim scores:

    h -> layer_norm -> linear(gelu) -> linear(+ h) -> layer_norm -> linear -> unit length

Queries are noisy copies of some tokens of their own document; the loss is cross
entropy over the batch's documents (in-batch negatives), so gradients run from
flash_maxsim_train_batched through the head into AdamW. Weights are bfloat16:
with --bits 32 they are copies that the optimizer writes of its float32
parameters, with --bits 8 the parameters themselves, with 8-bit moments.

    python examples/train_token_head.py [--steps 30] [--bits 8]
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import flash_maxsim_amd as fm  # noqa: E402


class TokenHead:
    """Weights of the head and its forward pass, in bfloat16."""

    def __init__(self, hidden: int, inner: int, d: int, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(n, k):
            return torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)

        def vector(n, value):
            return torch.full((n,), float(value), device="cuda")

        self.master = {
            "norm1.w": vector(hidden, 1), "norm1.b": vector(hidden, 0),
            "up.w": matrix(inner, hidden), "up.b": vector(inner, 0),
            "down.w": matrix(hidden, inner), "down.b": vector(hidden, 0),
            "norm2.w": vector(hidden, 1), "norm2.b": vector(hidden, 0),
            "out.w": matrix(d, hidden), "out.b": vector(d, 0),
        }
        self.w = {k: v.bfloat16().requires_grad_(True) for k, v in self.master.items()}

    def __call__(self, h: torch.Tensor) -> torch.Tensor:
        """Unit token embeddings [..., d] of hidden states [..., hidden]."""
        w = self.w
        x = fm.layer_norm(h, w["norm1.w"], w["norm1.b"])
        x = fm.linear(x, w["up.w"], w["up.b"], "gelu")
        x = fm.linear(x, w["down.w"], w["down.b"], residual=h)
        x = fm.layer_norm(x, w["norm2.w"], w["norm2.b"])
        return F.normalize(fm.linear(x, w["out.w"], w["out.b"]).float(), dim=-1).bfloat16()


def train(steps: int = 30, bits: int = 32, batch: int = 16, Lq: int = 32, Ld: int = 180, hidden: int = 256,
          inner: int = 1024, d: int = 128, lr: float = 1e-3, seed: int = 0) -> list[float]:
    """Losses of the steps."""
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    head = TokenHead(hidden, inner, d, seed)
    names = list(head.w)
    if bits == 8:
        opt = fm.AdamW(head.w.values(), lr=lr, state_bits=8)
    else:
        moments = [fm.adamw_state(head.master[k]) for k in names]
    losses = []
    for step in range(1, steps + 1):
        docs = torch.randn(batch, Ld, hidden, generator=g, device="cuda")
        lengths = torch.randint(Lq, Ld + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
        pick = (torch.rand(batch, Lq, generator=g, device="cuda") * lengths[:, None]).long()
        queries = docs.gather(1, pick[:, :, None].expand(-1, -1, hidden))
        queries = queries + 2.0 * torch.randn(queries.shape, generator=g, device="cuda")

        scores = fm.flash_maxsim_train_batched(head(queries.bfloat16()), head(docs.bfloat16()), lengths)
        loss = F.cross_entropy(scores, torch.arange(batch, device="cuda"))
        grads = torch.autograd.grad(loss, [head.w[k] for k in names])
        # the gradients' length is kept to one; the factor stays on the GPU
        clip = torch.clamp(1.0 / torch.linalg.vector_norm(torch.stack([x.float().norm() for x in grads])), max=1.0)
        if bits == 8:
            for k, x in zip(names, grads):
                head.w[k].grad = x
            opt.step(grad_scale=clip)
        else:
            fm.adamw_step([head.master[k] for k in names], grads, [m for m, _ in moments], [v for _, v in moments],
                          step, lr=lr, grad_scale=clip, copies=[head.w[k] for k in names])
        losses.append(float(loss.detach()))
    return losses


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--bits", type=int, choices=(8, 32), default=32)
    a = ap.parse_args()
    losses = train(a.steps, a.bits)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i + 1:4d}  loss {losses[i]:.4f}")
    print(f"last       loss {losses[-1]:.4f}")


if __name__ == "__main__":
    main()
