"""The norms' rings of rows: many more rows than the rings hold give, bit for bit, what few rows give,
where no slot is filled a second time. Rows of up to 512 elements belong to one warp each."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops

pytestmark = pytest.mark.gpu

# 296 CTAs of eight rows and up to eight stages hold 18944 rows under way; pieces of 1500 rows
# give a group one row at most.
ROWS, PIECE = 40000, 1500


def inputs(device, columns, dtype, count):
    gen = torch.Generator(device=device).manual_seed(columns)
    return [torch.randn(ROWS, columns, generator=gen, device=device).to(dtype) for _ in range(count)]


def pieces():
    return [slice(a, a + PIECE) for a in (0, 18000, ROWS - PIECE)]


@pytest.mark.parametrize("columns", [24, 250, 256, 505, 512, 1000, 1024])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rms_norm(cuda_device, columns, dtype):
    x, residual, grad, grad_total = inputs(cuda_device, columns, dtype, 4)
    weight = torch.rand(columns, device=cuda_device) + 0.5
    y, total, rstd = ops.rms_norm(x, weight, residual)
    codes, scales, _, _ = ops.rms_norm_8bit(x, weight, residual)
    dx, _ = ops.rms_norm_backward(grad, total, weight, rstd, grad_total)
    for _ in range(3):
        assert torch.equal(ops.rms_norm_backward(grad, total, weight, rstd, grad_total)[0], dx)
    for part in pieces():
        want = ops.rms_norm(x[part], weight, residual[part])
        for a, b in zip((y, total, rstd), want):
            assert torch.equal(a[part], b)
        want8 = ops.rms_norm_8bit(x[part], weight, residual[part])
        assert torch.equal(codes[part].float(), want8[0].float()) and torch.equal(scales[part], want8[1])
        alone, _ = ops.rms_norm_backward(grad[part], total[part], weight, rstd[part], grad_total[part])
        assert torch.equal(dx[part], alone)
