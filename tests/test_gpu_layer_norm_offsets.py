"""Layer norm of rows whose mean is large beside their deviations."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("columns", [64, 500, 513, 1000, 1024, 4096, 5001, 16384, 20000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("value", [3.0, -96.0, 416.0])
def test_constant_rows_give_the_bias(cuda_device, columns, dtype, value):
    """The sum of up to 2^24 / 416 equal whole numbers below 417 is exact in fp32, so the sum of a
    row is. Its mean is then one rounding of 1 / columns and one of the product off at most:
    |x - mean| <= 2^-23 |x|, and the result that far times rstd = eps^-1/2 = 316.3 (and not more)
    from the bias; exactly the bias where the number of columns is a power of two."""
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    x = torch.full((5, columns), value, dtype=dtype, device=cuda_device)
    weight = 1 + 0.1 * torch.randn(columns, generator=gen, device=cuda_device)
    bias = torch.randn(columns, generator=gen, device=cuda_device)
    epsilon = 1e-5
    y, mean, _ = ops.layer_norm(x, weight, bias, epsilon)
    error = 0.0 if columns & (columns - 1) == 0 else 2.0**-23 * abs(value) * 316.3 * weight.double().abs()
    if not columns & (columns - 1):
        assert (mean == value).all()
    rounding = torch.finfo(dtype).eps / 2 * (bias.double().abs() + error) + (2.0**-25 if dtype == torch.float16 else 0.0)
    assert ((y.double() - bias.double()).abs() <= error + rounding).all()
