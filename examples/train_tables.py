"""Train the parts that a LoRA run leaves frozen: a token table, layer norms and a vocabulary projection.

    python examples/train_tables.py [--device cuda] [--steps 40] [--vocab 4096] [--hidden 256]

A small residual model learns the successor of each token on padded synthetic
sequences.  One step runs the framework's operators as a training loop uses them:

* ``embedding`` looks the tokens up (scaled; the padding row gets no gradient),
* ``layer_norm`` before the block and before the head,
* ``linear_cross_entropy`` gives the loss of the answers (padding and prompt are
  ignored) and the gradients of the hidden states and of the projection,
* ``clip_grad_norm_`` clips all gradients by their global norm into the
  optimizer's fp32 buffer,
* ``FlatAdamW`` updates the fp32 masters, which are copied back to the model's type.
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from graspo_b200.engine.optim import FlatAdamW  # noqa: E402
from graspo_b200.ops.cross_entropy import linear_cross_entropy  # noqa: E402
from graspo_b200.ops.embedding import embedding  # noqa: E402
from graspo_b200.ops.grad_clip import clip_grad_norm_  # noqa: E402
from graspo_b200.ops.layer_norm import layer_norm  # noqa: E402

IGNORE = -100


class FlatParameters:
    """The model's tensors, their fp32 masters and gradients in two flat buffers
    (what ``FlatAdamW`` updates)."""

    replicated_numel = 0

    def __init__(self, tensors: list[torch.Tensor]) -> None:
        self.tensors = tensors
        sizes = [t.numel() for t in tensors]
        self.params = torch.cat([t.detach().float().reshape(-1) for t in tensors])
        self.grads = torch.zeros_like(self.params)
        self.masters = [m.view(t.shape) for m, t in zip(self.params.split(sizes), tensors)]
        self.views = [g.view(t.shape) for g, t in zip(self.grads.split(sizes), tensors)]

    def invalidate(self) -> None:
        with torch.no_grad():
            for t, master in zip(self.tensors, self.masters):
                t.copy_(master)


class SuccessorModel:
    def __init__(self, vocab: int, hidden: int, device: torch.device, dtype: torch.dtype, seed: int) -> None:
        g = torch.Generator().manual_seed(seed)

        def weight(*shape: int, std: float) -> torch.Tensor:
            return (torch.randn(*shape, generator=g) * std).to(device, dtype).requires_grad_(True)

        self.scale = math.sqrt(hidden)
        self.pad = vocab - 1
        self.table = weight(vocab, hidden, std=1 / self.scale)
        self.norms = [(torch.ones(hidden, device=device, dtype=dtype, requires_grad=True),
                       torch.zeros(hidden, device=device, dtype=dtype, requires_grad=True)) for _ in range(2)]
        self.up = weight(4 * hidden, hidden, std=1 / math.sqrt(hidden))
        self.down = weight(hidden, 4 * hidden, std=0.5 / math.sqrt(4 * hidden))
        self.head = weight(vocab, hidden, std=0.5 / math.sqrt(hidden))
        self.tensors = [self.table, *(t for n in self.norms for t in n), self.up, self.down, self.head]

    def loss(self, ids: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        x = embedding(ids, self.table, scale=self.scale, padding_idx=self.pad)
        x = x + F.linear(F.gelu(F.linear(layer_norm(x, *self.norms[0]), self.up)), self.down)
        return linear_cross_entropy(layer_norm(x, *self.norms[1]), self.head, targets, ignore_index=IGNORE)


def batch(vocab: int, rows: int, length: int, pad: int, g: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """Left-padded sequences of a fixed successor rule; the first quarter of each is a prompt."""
    words = min(vocab - 1, 64)
    seq = torch.randint(0, words, (rows, 1), generator=g)
    for _ in range(length):
        seq = torch.cat([seq, (5 * seq[:, -1:] + 17) % words], 1)
    ids, targets = seq[:, :-1].clone(), seq[:, 1:].clone()
    start = torch.randint(0, length // 2, (rows, 1), generator=g)
    at = torch.arange(length)[None]
    ids[at < start] = pad
    targets[at < start + length // 4] = IGNORE
    return ids, targets


def train(*, steps: int, vocab: int, hidden: int, rows: int = 8, length: int = 32, lr: float = 3e-3,
          max_norm: float = 1.0, device: str = "cuda", seed: int = 0, log=print) -> list[float]:
    dev = torch.device(device)
    model = SuccessorModel(vocab, hidden, dev, torch.bfloat16 if dev.type == "cuda" else torch.float32, seed)
    flat = FlatParameters(model.tensors)
    optim = FlatAdamW(flat, lr=lr, weight_decay=0.0)
    g = torch.Generator().manual_seed(seed + 1)
    losses = []
    for step in range(steps):
        ids, targets = (t.to(dev) for t in batch(vocab, rows, length, model.pad, g))
        loss = model.loss(ids, targets)
        grads = torch.autograd.grad(loss, model.tensors)
        norm = clip_grad_norm_(grads, max_norm, out=flat.views)
        optim.step(0.0, loss.detach().reshape(1))          # clipped already
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step == steps - 1:
            log(f"step {step}: loss {losses[-1]:.4f}, gradient norm {float(norm):.3f}")
    if dev.type == "cuda":
        from graspo_b200.ops._ext import check_errors

        check_errors()
    return losses


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--vocab", type=int, default=4096)
    ap.add_argument("--hidden", type=int, default=256)
    a = ap.parse_args()
    train(steps=a.steps, vocab=a.vocab, hidden=a.hidden, device=a.device)


if __name__ == "__main__":
    main()
