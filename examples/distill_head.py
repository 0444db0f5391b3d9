"""Distils the output end of a language model with the operators of this package.

    python -m examples.distill_head [--steps 60] [--width 512] [--vocabulary 8000]

The student's end: the last layer's output is added to the residual stream, normed, and
multiplied by the vocabulary's matrix, the norm and the matrix in 8 bits with scales for
blocks of 128. A fixed random end of the same kind teaches it by its top logits. The matrix
is stepped by Muon, the norm's weight by AdamW with 8-bit moments. Some tokens of each batch
stand for a prompt and have no part in the loss.
"""

from __future__ import annotations

import argparse

import torch
from torch import Tensor, nn

from gram_newton_schulz_ampere_b200 import Muon
from gram_newton_schulz_ampere_b200.training import distillation_loss, rms_norm_linear_8bit


class Head(nn.Module):
    def __init__(self, width: int, vocabulary: int, device: torch.device) -> None:
        super().__init__()
        self.norm = nn.Parameter(torch.ones(width, device=device))
        self.matrix = nn.Parameter(torch.randn(vocabulary, width, device=device, dtype=torch.bfloat16) * 4 * width**-0.5)

    def forward(self, x: Tensor, stream: Tensor) -> Tensor:
        return rms_norm_linear_8bit(x, self.norm, self.matrix, stream)[0]


def train(steps: int = 60, width: int = 512, vocabulary: int = 8000, tokens: int = 1024, top: int = 32,
          temperature: float = 2.0, seed: int = 0) -> list[float]:
    """The loss of each step."""
    device = torch.device("cuda")
    torch.manual_seed(seed)
    teacher, student = (Head(width, vocabulary, device) for _ in range(2))
    optimizer = Muon(
        [
            {"params": [student.matrix]},
            {"params": [student.norm], "algorithm": "adamw", "lr": 3e-3, "state_bits": 8, "state_rounding": "unbiased"},
        ],
        lr=0.02,
    )
    losses = []
    for _ in range(steps):
        x, stream = (torch.randn(tokens, width, device=device).bfloat16() for _ in range(2))
        answered = torch.rand(tokens, device=device) < 0.8
        with torch.no_grad():
            values, indices = teacher(x, stream).topk(top)
            indices = torch.where(answered[:, None], indices, -1)
        rows = distillation_loss(student(x, stream), indices, values, temperature)
        loss = rows.sum() / answered.sum()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--width", type=int, default=512)
    parser.add_argument("--vocabulary", type=int, default=8000)
    args = parser.parse_args()
    history = train(args.steps, args.width, args.vocabulary)
    for step in range(0, len(history), max(1, len(history) // 10)):
        print(f"step {step:4d}  loss {history[step]:.4f}")
    print(f"last       loss {history[-1]:.4f}")
