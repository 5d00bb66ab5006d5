"""Trains a small token encoder, from ids to MaxSim, on synthetic documents.

    ids -> embedding -> layer_norm -> blocks -> linear -> unit length
    block: gated_linear -> linear, then residual_norm adds it, normalised and scaled, to the hidden states and
           normalises them for the next block

Queries are some tokens of their own document, some of them replaced by random ones; the loss is cross entropy over the
batch's documents (in-batch negatives), so gradients run from flash_maxsim_train_batched through all layers into two
optimizers: Muon moves the blocks' matrices, AdamW the table, the vectors and the projection. Both keep float32
parameters and write the bfloat16 copies that the next forward pass reads.

    python examples/train_encoder_block.py [--steps 30]
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


class TokenEncoder:
    """Weights of the encoder and its forward pass, in bfloat16; id 0 is padding."""

    def __init__(self, vocabulary: int, hidden: int, inner: int, blocks: int, d: int, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(n, k):
            return torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)

        def vector(n, value):
            return torch.full((n,), float(value), device="cuda")

        self.blocks, self.hidden = blocks, hidden
        self.master = {"table": matrix(vocabulary, hidden), "norm.w": vector(hidden, 1), "norm.b": vector(hidden, 0)}
        for i in range(blocks):
            self.master |= {f"{i}.gate": matrix(inner, hidden), f"{i}.up": matrix(inner, hidden),
                            f"{i}.down": matrix(hidden, inner), f"{i}.post": vector(hidden, 1),
                            f"{i}.scale": vector(hidden, 0.5), f"{i}.norm": vector(hidden, 1)}
        self.master |= {"out.w": matrix(d, hidden), "out.b": vector(d, 0)}
        self.w = {k: v.bfloat16().requires_grad_(True) for k, v in self.master.items()}
        self.matrices = [k for k in self.w if k.split(".")[-1] in ("gate", "up", "down")]

    def __call__(self, ids: torch.Tensor) -> torch.Tensor:
        """Unit token embeddings [..., d] of ids [...]."""
        w = self.w
        h = fm.embedding(ids, w["table"], scale=math.sqrt(self.hidden), padding_idx=0)
        x = fm.layer_norm(h, w["norm.w"], w["norm.b"])
        for i in range(self.blocks):
            f = fm.linear(fm.gated_linear(x, w[f"{i}.gate"], w[f"{i}.up"], activation="silu"), w[f"{i}.down"])
            h, x = fm.residual_norm(f, h, w[f"{i}.norm"], norm="rms", post_norm=True, post_weight=w[f"{i}.post"],
                                    scale=w[f"{i}.scale"])
        return F.normalize(fm.linear(x, w["out.w"], w["out.b"]).float(), dim=-1).bfloat16()


def train(steps: int = 30, batch: int = 16, Lq: int = 32, Ld: int = 180, vocabulary: int = 5000, hidden: int = 256,
          inner: int = 512, blocks: int = 2, d: int = 128, seed: int = 0) -> list[float]:
    """Losses of the steps."""
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    model = TokenEncoder(vocabulary, hidden, inner, blocks, d, seed)
    for k, p in model.master.items():
        p.requires_grad_(True)
    others = [k for k in model.w if k not in model.matrices]
    muon = fm.Muon([model.master[k] for k in model.matrices], lr=0.02, copies=[model.w[k] for k in model.matrices])
    adamw = fm.AdamW([model.master[k] for k in others], lr=1e-3, copies=[model.w[k] for k in others])
    losses = []
    for _ in range(steps):
        lengths = torch.randint(Lq, Ld + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
        docs = torch.randint(1, vocabulary, (batch, Ld), generator=g, device="cuda")
        docs = docs * (torch.arange(Ld, device="cuda") < lengths[:, None])
        pick = (torch.rand(batch, Lq, generator=g, device="cuda") * lengths[:, None]).long()
        noise = torch.randint(1, vocabulary, (batch, Lq), generator=g, device="cuda")
        queries = torch.where(torch.rand(batch, Lq, generator=g, device="cuda") < 0.9, noise, docs.gather(1, pick))

        scores = fm.flash_maxsim_train_batched(model(queries), model(docs), lengths)
        loss = F.cross_entropy(scores, torch.arange(batch, device="cuda"))
        names = list(model.w)
        for k, x in zip(names, torch.autograd.grad(loss, [model.w[k] for k in names])):
            model.master[k].grad = x.float()
        muon.step()
        adamw.step()
        losses.append(float(loss.detach()))
    return losses


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    losses = train(ap.parse_args().steps)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i + 1:4d}  loss {losses[i]:.4f}")
    print(f"last       loss {losses[-1]:.4f}")


if __name__ == "__main__":
    main()
