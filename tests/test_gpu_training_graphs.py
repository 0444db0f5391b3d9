"""The training operators inside captured CUDA graphs and compiled regions."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops
from gram_newton_schulz_ampere_b200.training import grouped_linear, layer_norm

pytestmark = pytest.mark.gpu


def block(device, width=200, hidden=129, experts=4):
    gen = torch.Generator(device=device).manual_seed(1)

    def leaf(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=gen, device=device) * scale).to(dtype).requires_grad_()

    x = leaf(300, width)
    norm = leaf(width, dtype=torch.float32), leaf(width, dtype=torch.float32)
    weight = leaf(experts, hidden, width, scale=0.1)
    ends = torch.tensor([100, 100, 250, 290], device=device)
    return x, norm, weight, ends


def test_captured_forward_and_backward(cuda_device):
    """Odd sizes, so that the aligning copies are in the graph too; other inputs and other ends
    at the replay."""
    x, norm, weight, ends = block(cuda_device)
    grad = torch.randn(300, 129, device=cuda_device).bfloat16()

    def step():
        y = grouped_linear(layer_norm(x, *norm), weight, ends)
        return (y, *torch.autograd.grad(y, (x, *norm, weight), grad))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
        weight.mul_(0.5)
    ends.copy_(torch.tensor([0, 30, 280, 300], device=cuda_device))
    for _ in range(2):
        graph.replay()
    for got, want in zip(captured, step()):
        assert torch.equal(got, want)


def test_captured_adamw_step(cuda_device):
    """A captured step repeats the step number that it was captured with."""
    sizes = [5000, 33]
    params = [torch.ones(n, device=cuda_device) for n in sizes]
    twin = [p.clone() for p in params]
    grads = [torch.randn(n, device=cuda_device) for n in sizes]
    held, eager = ops.AdamWStates(params), ops.AdamWStates(twin)
    hyper = (1e-2, 0.9, 0.95, 1e-8, 0.1)
    held.step(grads, *hyper, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held.step(grads, *hyper, 7)
    graph.replay()
    eager.step(grads, *hyper, 1)
    eager.step(grads, *hyper, 7)
    assert all(torch.equal(p, q) for p, q in zip(params, twin))


def test_compiled_region_breaks_at_the_layers(cuda_device):
    x, norm, weight, ends = block(cuda_device)

    def loss(x):
        return grouped_linear(layer_norm(x, *norm) * 2, weight, ends).float().square().sum()

    want = torch.autograd.grad(loss(x), (x, *norm, weight))
    got = torch.autograd.grad(torch.compile(loss)(x), (x, *norm, weight))
    # fp32 elementwise work between the layers may be fused: a few roundings of bfloat16.
    for a, b in zip(got, want):
        assert torch.allclose(a.float(), b.float(), rtol=2.0**-6, atol=2.0**-6 * b.float().abs().max().item())


def test_types_under_autocast(cuda_device):
    """The layers do not cast: what comes in fp32 is refused or stays fp32."""
    x, norm, weight, ends = block(cuda_device)
    with torch.autocast("cuda", torch.bfloat16):
        assert layer_norm(x.float(), *norm).dtype == torch.float32
        assert grouped_linear(x, weight, ends).dtype == torch.bfloat16
        with pytest.raises(TypeError, match="float16 or bfloat16"):
            grouped_linear(x.float(), weight, ends)
