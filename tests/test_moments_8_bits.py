"""Moments brought into the 8-bit form and out of it, on the CPU."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops


@pytest.mark.parametrize("shape", [(), (0,), (1,), (255,), (256,), (257,), (3, 100)])
@pytest.mark.parametrize("second", [False, True])
def test_there_and_back(shape, second):
    gen = torch.Generator().manual_seed(1)
    values = torch.randn(shape, generator=gen) * 10 ** (3 * torch.randn(shape, generator=gen))
    if second:
        values = values.abs()
    codes, scales = ops.moment_in_8_bits(values, second)
    assert codes.shape == values.shape and codes.dtype == torch.float8_e4m3fn and codes.is_contiguous()
    assert scales.shape == ((values.numel() + 255) // 256,)
    back = ops.moment_from_8_bits(codes, scales)
    assert back.shape == values.shape and back.dtype == torch.float32
    smallest = scales.double().repeat_interleave(256)[:values.numel()].view(shape) * (2.0**-9 if second else 2.0**-10)
    bound = torch.maximum(values.double().abs() * 2.0**-4, smallest) * (1 + 2.0**-20)
    assert ((back.double() - values.double()).abs() <= bound).all()
    if second:
        assert (back[values > 0] > 0).all()


def test_zeros_and_what_is_not_finite():
    codes, scales = ops.moment_in_8_bits(torch.zeros(300), True)
    assert not codes.float().any() and not scales.any()
    values = torch.ones(600)
    values[10] = float("nan")
    values[300] = float("inf")
    back = ops.moment_from_8_bits(*ops.moment_in_8_bits(values, False))
    assert not back[:512].isfinite().any() and (back[512:] == 1).all()
