"""The differentiable layers, Muon's AdamW groups with held moments, and the example that runs them together."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

from gram_newton_schulz_ampere_b200 import Muon, ops
from gram_newton_schulz_ampere_b200.training import grouped_linear, layer_norm

pytestmark = pytest.mark.gpu


def test_layer_norm_gradient_against_differences(cuda_device):
    """Central differences of the fp32 operator along random directions. With steps of 2^-7 the
    third-order term and the rounding of a sum of 600 terms of size one are both near 1e-3
    of the sum of magnitudes; the bound is 1e-2 of it."""
    gen = torch.Generator(device=cuda_device).manual_seed(1)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=cuda_device)

    x, w, b, dy = normal(6, 100), 1 + 0.1 * normal(100), normal(100), normal(6, 100)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    layer_norm(*leaves).backward(dy)
    for i, leaf in enumerate(leaves):
        direction = normal(*leaf.shape)
        step = 2.0**-7

        def value(sign):
            inputs = [t.clone() for t in (x, w, b)]
            inputs[i] = inputs[i] + sign * step * direction
            return (layer_norm(*inputs).double() * dy.double()).sum()

        slope = (value(1) - value(-1)) / (2 * step)
        products = leaf.grad.double() * direction.double()
        assert abs((slope - products.sum()).item()) <= 1e-2 * products.abs().sum().item()


def test_grouped_linear_gradient(cuda_device):
    """Both gradients against autograd through 64-bit products: one rounding to bfloat16
    (2^-8) and fp32 sums of at most 96 terms."""
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    counts = [40, 0, 96, 7]
    rows = sum(counts) + 3
    x = torch.randn(rows, 72, generator=gen, device=cuda_device).bfloat16().requires_grad_()
    w = (torch.randn(4, 88, 72, generator=gen, device=cuda_device) * 0.1).bfloat16().requires_grad_()
    dy = torch.randn(rows, 88, generator=gen, device=cuda_device).bfloat16()
    ends = torch.tensor(counts, device=cuda_device).cumsum(0)
    grouped_linear(x, w, ends).backward(dy)
    x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    parts, at = [], 0
    for e, n in enumerate(counts):
        parts.append(x64[at:at + n] @ w64[e].T)
        at += n
    torch.cat(parts).backward(dy[:at].double())
    for got, want in ((x.grad, x64.grad), (w.grad, w64.grad)):
        size = want.abs().max()
        assert ((got.double() - want).abs() <= 2.0**-8 * want.abs() + 96 * 2.0**-23 * 96 * size).all()
    assert not x.grad[sum(counts):].any() and not w.grad[1].any()


def test_gradients_only_where_needed(cuda_device):
    x = torch.randn(8, 64, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(2, 32, 64, device=cuda_device, dtype=torch.bfloat16)
    ends = torch.tensor([3, 8], device=cuda_device)
    y = grouped_linear(x, w, ends)
    assert y.requires_grad and not grouped_linear(x.detach(), w, ends).requires_grad
    y.sum().backward()  # an expanded gradient, with zero strides
    assert x.grad is not None and w.grad is None
    n = torch.ones(64, device=cuda_device, requires_grad=True)
    layer_norm(x.detach(), n).sum().backward()
    assert n.grad is not None
    with pytest.raises(ValueError, match="experts, out, in"):
        grouped_linear(x, w[0], ends)


@pytest.mark.parametrize("bits", [8, 32])
def test_muon_adamw_group_with_held_moments(cuda_device, bits):
    """A group steps as AdamWStates does, parameters without a gradient stay, and a saved and
    loaded optimizer goes on with the same bits."""
    torch.manual_seed(3)

    def make():
        return [torch.nn.Parameter(torch.linspace(-1, 1, n, device=cuda_device).bfloat16()) for n in (700, 33, 256)]

    ours, twin = make(), make()
    ours[2].data = ours[2].data.view(16, 16).T  # not contiguous
    optimizer = Muon([{"params": ours, "algorithm": "adamw", "state_bits": bits}], lr=1e-2, weight_decay=0.1)
    twin[2].data = twin[2].data.view(16, 16).T.contiguous()
    states = ops.AdamWStates([p.data for p in twin], bits)

    def step(opt, params, number):
        grads = [torch.randn(p.shape, device=cuda_device).bfloat16() for p in params]
        for p, g in zip(params, grads):
            p.grad = g
        if number == 2:
            params[1].grad = None
            grads[1] = None
        opt.step()
        return grads

    counts = [0, 0, 0]
    for number in (1, 2, 3):
        grads = step(optimizer, ours, number)
        counts = [c + (g is not None) for c, g in zip(counts, grads)]
        states.step(grads, 1e-2, 0.9, 0.95, 1e-8, 0.1, [max(c, 1) for c in counts])
    for p, q in zip(ours, twin):
        assert torch.equal(p, q)
    expected = torch.float8_e4m3fn if bits == 8 else torch.float32
    assert optimizer.state[ours[0]]["exp_avg"].dtype == expected

    copies = make()
    for c, p in zip(copies, ours):
        c.data = p.data.clone()
    second = Muon([{"params": copies, "algorithm": "adamw", "state_bits": bits}], lr=1e-2, weight_decay=0.1)
    second.load_state_dict(optimizer.state_dict())
    for p, c in zip(ours, copies):
        for name, value in optimizer.state[p].items():
            assert second.state[c][name].dtype == value.dtype and torch.equal(second.state[c][name].float(), value.float())
    torch.manual_seed(4)
    step(optimizer, ours, 4)
    torch.manual_seed(4)
    step(second, copies, 4)
    for p, c in zip(ours, copies):
        assert torch.equal(p, c)


def test_muon_refuses_state_bits(cuda_device):
    vector = torch.nn.Parameter(torch.ones(8, device=cuda_device))
    matrix = torch.nn.Parameter(torch.ones(8, 8, device=cuda_device))
    with pytest.raises(ValueError, match="state_bits must be"):
        Muon([{"params": [vector], "algorithm": "adamw", "state_bits": 4}])
    with pytest.raises(ValueError, match="adamw groups"):
        Muon([{"params": [matrix], "state_bits": 8}])


def test_example_learns(cuda_device):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    try:
        import train_expert_block
    finally:
        sys.path.pop(0)
    losses = train_expert_block.train(steps=30, width=128, experts=4, tokens=512)
    assert all(loss == loss for loss in losses)
    assert sum(losses[-5:]) < 0.8 * sum(losses[:5])
