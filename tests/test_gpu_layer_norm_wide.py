"""Rows at the limits of the ring, and rows that no ring holds, more of them than CTAs."""

from __future__ import annotations

import pytest
import torch

from test_gpu_layer_norm import check_norm, inputs

pytestmark = pytest.mark.gpu


# In fp32 a stage of x and dy fits the 200 KB ring twice up to 12800 elements; rows of
# more than 16384 have no ring in either pass. A device has 148 SMs, two CTAs on each.
@pytest.mark.parametrize("columns", [12792, 12800, 12801, 12804, 14336, 16383, 16384, 16385, 20001])
@pytest.mark.parametrize("rows", [1, 299, 650])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm(cuda_device, rows, columns, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    check_norm(*inputs(gen, rows, columns, dtype, torch.float32, cuda_device))


@pytest.mark.parametrize("columns", [12797, 14336, 17001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_that_start_anywhere(cuda_device, columns, dtype):
    """Between rows of NaN, x and its gradient at different offsets."""
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    values, weight, bias, grads = inputs(gen, 301, columns, dtype, torch.float32, cuda_device)
    wide = torch.full((303, columns + 6), float("nan"), dtype=dtype, device=cuda_device)
    grad = torch.full((303, columns + 11), float("nan"), dtype=dtype, device=cuda_device)
    x, dy = wide[1:-1, 1:columns + 1], grad[1:-1, 3:columns + 3]
    x.copy_(values)
    dy.copy_(grads)
    check_norm(x, weight, bias, dy)
