"""The output end's operators where element offsets pass 32 bits, and inside compiled regions."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops
from gram_newton_schulz_ampere_b200.training import distillation_loss, rms_norm_linear_8bit

pytestmark = pytest.mark.gpu

BLOCK = 128


def filled(rows, columns, device, dtype=torch.bfloat16):
    """Rows that repeat every 1000, without a 32-bit copy of the whole."""
    some = torch.randn(1000, columns, device=device).to(dtype)
    whole = torch.empty(rows, columns, dtype=dtype, device=device)
    for a in range(0, rows, 1000):
        whole[a:a + 1000] = some[: min(1000, rows - a)]
    return whole


def test_many_rows(cuda_device):
    """600001 rows of 4096: the last ones give what they give by themselves."""
    x = filled(600001, 4096, cuda_device)
    last = x[-300:].clone()
    codes, scales = ops.quantize_8bit(x)
    want, want_scales = ops.quantize_8bit(last)
    assert torch.equal(codes[-300:].view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales[-300:], want_scales)
    del codes, scales
    w = torch.randn(4096, device=cuda_device)
    eight = ops.rms_norm_8bit(x, w)
    for got, alone in zip(eight[:2], ops.rms_norm_8bit(last, w)[:2]):
        assert torch.equal(got[-300:].float(), alone.float())
    rstd = eight[3]
    del eight
    y, _, _ = ops.rms_norm(x, w, x)
    assert torch.equal(y[-300:], ops.rms_norm(last, w, last)[0])
    dx, _ = ops.rms_norm_backward(y, x, w, rstd)
    assert torch.equal(dx[-300:], ops.rms_norm_backward(y[-300:].clone(), last, w, rstd[-300:].clone())[0])


def test_large_product(cuda_device):
    """70000 x 200 x 32768: the last rows and columns, in a tile grid of 273 x 128."""
    x, w = torch.randn(70000, 200, device=cuda_device), torch.randn(32768, 200, device=cuda_device)
    xc, xs = ops.quantize_8bit(x)
    wc, ws = ops.quantize_8bit(w, BLOCK)
    out = ops.gemm_8bit(xc, xs, wc.t(), ws.t())
    part = ops.gemm_8bit(xc[-600:], xs[-600:], wc[-512:].t(), ws[-4:].t(), out_dtype=torch.float32)
    # Other tiles, and so other roundings of the same sums, at most half a step of bfloat16 and an ulp of fp32.
    off = (out[-600:, -512:].float() - part).abs()
    assert (off <= 2.0**-8 * part.abs() + 200 * 2.0**-22 * part.abs().amax()).all()


def test_large_logits_tensor(cuda_device):
    rows, vocabulary = 17001, 131072
    logits = filled(rows, vocabulary, cuda_device)
    indices = torch.randint(0, vocabulary, (rows, 8), device=cuda_device)
    teacher = torch.randn(rows, 8, device=cuda_device)
    grad = torch.rand(rows, device=cuda_device)
    loss, dlogits = ops.distillation_loss_gradient(grad, logits, indices, teacher)
    # As many rows that each has an SM to itself here too: the same order of sums.
    tail = slice(rows - 400, rows)
    want, want_dlogits = ops.distillation_loss_gradient(grad[tail], logits[tail].clone(), indices[tail], teacher[tail])
    assert torch.equal(loss[tail], want) and torch.equal(dlogits[tail], want_dlogits)


def test_compiled_region_breaks_at_the_layers(cuda_device):
    def leaf(*shape):
        return torch.randn(shape, device=cuda_device).bfloat16().requires_grad_()

    x, stream, norm, head = leaf(64, 128), leaf(64, 128), leaf(128), leaf(300, 128)
    indices, teacher = torch.randint(0, 300, (64, 5), device=cuda_device), torch.randn(64, 5, device=cuda_device)

    def loss(x):
        logits, total = rms_norm_linear_8bit(x * 2, norm, head, stream)
        return distillation_loss(logits, indices, teacher).sum() + total.float().square().sum()

    leaves = (x, stream, norm, head)
    want = torch.autograd.grad(loss(x), leaves)
    got = torch.autograd.grad(torch.compile(loss)(x), leaves)
    # Elementwise work between the layers may be fused: a few roundings of bfloat16.
    for a, b in zip(got, want):
        assert torch.allclose(a.float(), b.float(), rtol=2.0**-6, atol=2.0**-6 * b.float().abs().max().item())
