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


@pytest.mark.parametrize("columns", [1, 5, 77, 505, 1111, 4093])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_what_lies_beside_the_rows_is_not_used(cuda_device, columns, dtype):
    """Rows of views at every place within 16 bytes, with NaN before, behind and between them, give what
    they give by themselves but for the order of sums: a step of the type and 2^-18 of a row's
    largest value (a few dozen roundings of 2^-24 in each statistic), in the gradient of the terms that
    it is the difference of."""
    gen = torch.Generator(device=cuda_device).manual_seed(columns)
    rows = 30
    weight, bias = torch.rand(columns, device=cuda_device) + 0.5, torch.randn(columns, device=cuda_device)

    def embedded(shift):
        t = torch.randn(rows, columns, generator=gen, device=cuda_device).to(dtype)
        wide = torch.full((rows, columns + 16), float("nan"), dtype=dtype, device=cuda_device)
        return t, wide[:, shift:shift + columns].copy_(t)

    def near(got, want, terms=None):
        size = want.double().abs()
        terms = size.amax(-1, keepdim=True) if terms is None else terms
        allowed = torch.finfo(dtype).eps * size + 2.0**-18 * terms + 2.0**-24
        assert torch.isfinite(got).all() and ((got.double() - want.double()).abs() <= allowed).all()

    for shift in range(8):
        (x, x_in), (r, r_in), (g, g_in), (s, s_in) = (embedded((shift + i) % 8 + 1) for i in range(4))
        y, total, rstd = ops.rms_norm(x_in, weight, r_in)
        want, want_total, _ = ops.rms_norm(x, weight, r)
        assert torch.equal(total, want_total)
        near(y, want)
        want, _, want_rstd = ops.rms_norm(x, weight)
        near(ops.rms_norm(x_in, weight)[0], want)
        assert torch.isfinite(ops.rms_norm_8bit(x_in, weight, r_in)[0].float()).all()
        dx, dweight = ops.rms_norm_backward(g_in, x_in, weight, want_rstd, s_in)
        want = ops.rms_norm_backward(g, x, weight, want_rstd, s)
        h, a = x.double() * want_rstd.double()[:, None], (g.double() * weight.double())
        terms = want_rstd.double()[:, None] * (a.abs() + h.abs() * (a * h).abs().mean(1, keepdim=True)) + s.double().abs()
        near(dx, want[0], terms)
        assert torch.isfinite(dweight).all()
        out, mean, rstd = ops.layer_norm(x_in, weight, bias, 1e-3)
        assert torch.isfinite(out).all()
        for t in ops.layer_norm_backward(g_in, x_in, weight, mean, rstd):
            assert torch.isfinite(t).all()
