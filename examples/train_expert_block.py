"""Trains a small pre-norm block of experts with the operators of this package.

    python -m examples.train_expert_block [--steps 60] [--width 256] [--experts 8]

One block: layer norm, a router that sends each token to one of the experts, and two linear
layers per expert. It learns to imitate a fixed random block. The experts' weights are
batches of matrices, stepped by Muon (one orthogonalisation per shape); the norm, router
and output scale are stepped by AdamW with 8-bit moments.
"""

from __future__ import annotations

import argparse

import torch
from torch import Tensor, nn

from gram_newton_schulz_ampere_b200 import Muon
from gram_newton_schulz_ampere_b200.training import grouped_linear, layer_norm


class ExpertBlock(nn.Module):
    def __init__(self, width: int, hidden: int, experts: int, device: torch.device) -> None:
        super().__init__()
        options = {"device": device, "dtype": torch.bfloat16}
        self.norm_weight = nn.Parameter(torch.ones(width, device=device))
        self.norm_bias = nn.Parameter(torch.zeros(width, device=device))
        self.router = nn.Parameter(torch.randn(experts, width, **options) * width**-0.5)
        self.up = nn.Parameter(torch.randn(experts, hidden, width, **options) * width**-0.5)
        self.down = nn.Parameter(torch.randn(experts, width, hidden, **options) * hidden**-0.5)

    def forward(self, x: Tensor) -> Tensor:
        h = layer_norm(x, self.norm_weight, self.norm_bias)
        gate, expert = torch.softmax((h @ self.router.T).float(), dim=-1).max(dim=-1)
        # Tokens in the order of their experts; the ends stay on the device.
        order = torch.argsort(expert, stable=True)
        ends = torch.bincount(expert, minlength=self.up.shape[0]).cumsum(0)
        rows = torch.nn.functional.gelu(grouped_linear(h[order], self.up, ends))
        rows = grouped_linear(rows, self.down, ends) * gate[order, None].to(x.dtype)
        return x + torch.zeros_like(x).index_copy(0, order, rows)


def train(steps: int = 60, width: int = 256, experts: int = 8, tokens: int = 2048, seed: int = 0) -> list[float]:
    """The loss of each step."""
    device = torch.device("cuda")
    torch.manual_seed(seed)
    teacher = ExpertBlock(width, 2 * width, experts, device)
    block = ExpertBlock(width, 2 * width, experts, device)
    optimizer = Muon(
        [
            {"params": [block.up, block.down]},
            {
                "params": [block.norm_weight, block.norm_bias, block.router],
                "algorithm": "adamw",
                "lr": 3e-3,
                "state_bits": 8,
                "state_rounding": "unbiased",
            },
        ],
        lr=0.01,
    )
    losses = []
    for _ in range(steps):
        x = torch.randn(tokens, width, device=device).bfloat16()
        with torch.no_grad():
            target = teacher(x)
        loss = (block(x) - target).float().square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--width", type=int, default=256)
    parser.add_argument("--experts", type=int, default=8)
    args = parser.parse_args()
    history = train(args.steps, args.width, args.experts)
    for step in range(0, len(history), max(1, len(history) // 10)):
        print(f"step {step:4d}  loss {history[step]:.4f}")
    print(f"last       loss {history[-1]:.4f}")
