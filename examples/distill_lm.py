"""Train a small language model with Muon, then distill it into a smaller one.

Both models are residual MLPs over a token embedding; the data is a noisy
permutation of the vocabulary (the next token follows from the last one with
probability 0.9). Hidden matrices are stepped by ``GroupedMuon``, embedding and
head by AdamW. The teacher learns by ``losses.linear_cross_entropy`` (prompt
tokens carry no loss), the student by ``losses.linear_distillation`` on the
teacher's top logits; both are scored token by token with ``reduction="none"``,
and the student's divergence once more from its logits by
``losses.distillation``.

    python examples/distill_lm.py [--steps 200] [--vocab 50257] [--dim 256]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from pytorch_opt_b200 import losses  # noqa: E402
from pytorch_opt_b200.muon import GroupedMuon, MuonGroup  # noqa: E402

IGNORE = -100


class Model:
    """Embedding, ``layers`` blocks x + silu(rms(x) A) B, head. bf16 matrices."""

    def __init__(self, vocab: int, dim: int, layers: int, device, seed: int):
        g = torch.Generator(device=device).manual_seed(seed)
        new = lambda std, *shape: (std * torch.randn(*shape, generator=g, device=device)).bfloat16()  # noqa: E731
        self.embed = new(1.0, vocab, dim).requires_grad_()
        self.head = new(0.02, vocab, dim).requires_grad_()
        self.blocks = new(dim**-0.5, 2 * layers, dim, dim).requires_grad_()

    @staticmethod
    def _rms(x):
        return x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6).to(x.dtype)

    def hidden(self, tokens):
        x = self.embed[tokens]
        for i in range(0, self.blocks.shape[0], 2):
            x = x + torch.nn.functional.silu(self._rms(x) @ self.blocks[i]) @ self.blocks[i + 1]
        return self._rms(x)


class Optimizer:
    """Muon for the blocks, AdamW for embedding and head."""

    def __init__(self, model: Model, lr: float):
        self.model = model
        self.blocks = MuonGroup(model.blocks.detach(), torch.zeros_like(model.blocks))
        self.muon = GroupedMuon([self.blocks], lr=0.02)
        self.adam = torch.optim.AdamW([model.embed, model.head], lr=lr)

    def step(self, loss) -> None:
        loss.backward()
        self.blocks.grads.copy_(self.model.blocks.grad)
        self.model.blocks.grad = None
        self.muon.step()
        self.adam.step()
        self.adam.zero_grad()


def batch(vocab: int, rows: int, length: int, g: torch.Generator, device):
    """Tokens (rows, length) and their targets, the first eighth of each row a prompt without loss."""
    x = torch.empty(rows, length + 1, dtype=torch.long, device=device)
    x[:, 0] = torch.randint(0, vocab, (rows,), generator=g, device=device)
    for i in range(length):
        x[:, i + 1] = (x[:, i] * 3 + 7) % vocab
        noise = torch.rand(rows, generator=g, device=device) < 0.1
        x[noise, i + 1] = torch.randint(0, vocab, (int(noise.sum()),), generator=g, device=device)
    target = x[:, 1:].clone()
    target[:, : length // 8] = IGNORE
    return x[:, :-1], target


def run(steps: int = 200, vocab: int = 50257, dim: int = 256, rows: int = 64, length: int = 64, top: int = 32,
        temperature: float = 2.0, say=print) -> dict:
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(1)
    out = {}

    teacher = Model(vocab, dim, 4, device, 0)
    opt = Optimizer(teacher, lr=1e-2)
    for i in range(steps):
        x, y = batch(vocab, rows, length, g, device)
        loss = losses.linear_cross_entropy(teacher.hidden(x), teacher.head, y, ignore_index=IGNORE, z_loss=1e-4)
        opt.step(loss)
        if i in (0, steps - 1):
            out["teacher first" if i == 0 else "teacher last"] = float(loss)

    student = Model(vocab, dim // 2, 2, device, 2)
    opt = Optimizer(student, lr=1e-2)
    for i in range(steps):
        x, y = batch(vocab, rows, length, g, device)
        with torch.no_grad():
            h = teacher.hidden(x)
            values, index = (h @ teacher.head.t()).topk(top, dim=-1)
            index[y == IGNORE] = -1
        loss = losses.linear_distillation(student.hidden(x), student.head, index, values, temperature=temperature)
        opt.step(loss)
        if i in (0, steps - 1):
            out["student first" if i == 0 else "student last"] = float(loss)

    with torch.no_grad():
        x, y = batch(vocab, rows, length, g, device)
        for name, m in (("teacher", teacher), ("student", student)):
            each = losses.linear_cross_entropy(m.hidden(x), m.head, y, ignore_index=IGNORE, reduction="none")
            out[name + " nats a token"] = float(each.sum() / (y != IGNORE).sum())
        values, index = (teacher.hidden(x) @ teacher.head.t()).topk(top, dim=-1)
        h = student.hidden(x)
        out["divergence, linear"] = float(losses.linear_distillation(h, student.head, index, values,
                                                                     temperature=temperature))
        out["divergence, logits"] = float(losses.distillation(h @ student.head.t(), index, values,
                                                              temperature=temperature))
    for k, v in out.items():
        say(f"{k:24s} {v:8.4f}")
    return out


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--vocab", type=int, default=50257)
    ap.add_argument("--dim", type=int, default=256)
    args = ap.parse_args()
    run(args.steps, args.vocab, args.dim)
    return 0


if __name__ == "__main__":
    sys.exit(main())
