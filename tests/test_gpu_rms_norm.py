"""RMS norm forward (with the residual's sum, in the stream's type and in 8 bits) and backward against 64 bits.

Bounds: a sum over a row takes at most 64 roundings on any path for rows of up to 65536 elements
(each thread's share, then a tree), so that rstd, half of the sum's error and the root's own, errs by
64 u r (u = 2^-24), an element h = t r by 64 u |h|; a sum over R rows by R u times the sum of
magnitudes. Results are rounded once to their type. The stream's sum is one fp32 addition rounded
once: torch's own."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops

pytestmark = pytest.mark.gpu

BLOCK, LEAST = 128, 448.0 * 2.0**-126
ROUNDING = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
U = 64 * 2.0**-24


def check(out, exact, error):
    absolute = 2.0**-25 if out.dtype == torch.float16 else 1e-40
    bound = error + ROUNDING[out.dtype] * (exact.abs() + error) + absolute
    worst = ((out.double() - exact).abs() - bound).max().item() if out.numel() else 0.0
    assert worst <= 0.0, f"largest excess {worst}"


def check_codes(codes, scales, y, error):
    """Scales within the error of a block's largest value and one rounding of the division, codes
    within half a step (2^-4 of the value, 2^-10 below 2^-6) and the error of what they code."""
    rows, columns = y.shape
    padded = torch.nn.functional.pad(y, (0, -columns % BLOCK)).view(rows, -1, BLOCK)
    wrong = torch.nn.functional.pad(error, (0, -columns % BLOCK)).view(rows, -1, BLOCK).amax(2)
    top = padded.abs().amax(2).clamp_min(LEAST)
    assert ((scales.double() - top / 448).abs() <= wrong / 448 + 2.0**-23 * top / 448).all()
    got = codes.double() * scales.double().repeat_interleave(BLOCK, 1)[:, :columns]
    step = scales.double().repeat_interleave(BLOCK, 1)[:, :columns]
    half = torch.maximum(2.0**-4 * y.abs(), 2.0**-10 * step)
    assert ((got - y).abs() <= half * (1 + 2.0**-18) + 2 * error + 2.0**-21 * y.abs()).all()


def check_norm(x, weight, residual, grad, grad_total, epsilon=1e-5):
    columns = weight.numel()
    y, total, rstd = ops.rms_norm(x, weight, residual, epsilon)
    codes, scales, total8, rstd8 = ops.rms_norm_8bit(x, weight, residual, epsilon)
    want_total = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    assert torch.equal(total, want_total) and torch.equal(total8, want_total)
    assert rstd.shape == x.shape[:-1] and torch.equal(rstd, rstd8)
    t64 = want_total.double().reshape(-1, columns)
    w64 = weight.double()
    r = 1 / (t64.square().mean(1, keepdim=True) + epsilon).sqrt()
    h = t64 * r
    check(rstd.reshape(-1, 1), r, U * r)
    check(y.reshape(-1, columns), h * w64, U * (h * w64).abs())
    check_codes(codes, scales, h * w64, U * (h * w64).abs())
    if grad is None:
        return
    dx, dweight = ops.rms_norm_backward(grad, total, weight, rstd, grad_total)
    assert dx.shape == x.shape and dx.dtype == x.dtype and dweight.dtype == weight.dtype
    dy = grad.double().reshape(-1, columns)
    a = dy * w64
    c, size = (a * h).mean(1, keepdim=True), (a * h).abs().mean(1, keepdim=True)
    want = r * (a - h * c)
    error = 4 * U * r * (a.abs() + h.abs() * size)
    if grad_total is not None:
        want = want + grad_total.double().reshape(-1, columns)
        error = error + 2.0**-24 * want.abs()
    check(dx.reshape(-1, columns), want, error)
    rows = max(t64.shape[0], 1)
    check(dweight, (dy * h).sum(0), (U + rows * 2.0**-24) * (dy * h).abs().sum(0))


def inputs(gen, rows, columns, dtype, w_dtype, device):
    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    x = (normal(rows, columns) * (0.5 + torch.rand((rows, 1), generator=gen, device=device)) + 0.3).to(dtype)
    return x, (1 + 0.2 * normal(columns)).to(w_dtype), *(normal(rows, columns).to(dtype) for _ in range(3))


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
         (torch.float32, torch.float32), (torch.float32, torch.bfloat16)]


@pytest.mark.parametrize("rows", [1, 5, 700])
@pytest.mark.parametrize("columns", [1, 2, 7, 64, 128, 136, 500, 512, 520, 1000, 1024, 1032, 1111, 2048, 4104, 8192, 9001])
@pytest.mark.parametrize("dtype,w_dtype", TYPES)
def test_norm(cuda_device, rows, columns, dtype, w_dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    x, weight, residual, grad, grad_total = inputs(gen, rows, columns, dtype, w_dtype, cuda_device)
    check_norm(x, weight, residual, grad, grad_total)
    check_norm(x, weight, None, grad, None)


@pytest.mark.parametrize("rows,columns", [(3, 16384), (3, 16385), (200, 16376), (70, 20000), (2, 40001), (4000, 96),
                                          (3, 12800), (3, 14336), (2000, 24), (5000, 1000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_of_long_and_many_rows(cuda_device, rows, columns, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    x, weight, residual, grad, grad_total = inputs(gen, rows, columns, dtype, torch.float32, cuda_device)
    check_norm(x, weight, residual, grad, grad_total)
    check_norm(x, weight, None, grad, None)
    check_norm(x, weight, residual, grad, None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("columns", [64, 640, 1111, 4096])
def test_norm_of_views(cuda_device, columns, dtype):
    """Rows that start anywhere, strided rows, other orders, more dimensions, each tensor its own."""
    gen = torch.Generator(device=cuda_device).manual_seed(3)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=cuda_device).to(dtype)

    weight = normal(columns + 3)[3:]
    for x, residual, grad, grad_total in (
        (normal(40, columns + 5)[:, 3:3 + columns], normal(40, columns), normal(40, columns + 8)[:, :columns], normal(40, columns)),
        (normal(40, columns)[::2], normal(20, columns + 1)[:, 1:], normal(columns, 20).t(), normal(1, columns).expand(20, columns)),
        (normal(3, 7, columns), normal(7, 3, columns).transpose(0, 1), normal(3, 7, columns), normal(3, 7, columns)),
    ):
        check_norm(x, weight, residual, grad, grad_total)


@pytest.mark.parametrize("columns", [100, 4096])
def test_extremes(cuda_device, columns):
    """Rows of zeros, of large and of tiny values, and with an infinity or a NaN, which stay in their rows."""
    x = torch.randn(6, columns, device=cuda_device)
    x[0] = 0.0
    x[1] *= 1e15
    x[2] *= 1e-15
    x[3, 3] = float("inf")
    x[4, 5] = float("nan")
    w = torch.ones(columns, device=cuda_device)
    good = [0, 1, 2, 5]
    y, _, rstd = ops.rms_norm(x, w)
    codes, scales, _, _ = ops.rms_norm_8bit(x, w)
    dx, _ = ops.rms_norm_backward(torch.ones_like(x), x, w, rstd)
    check_norm(x[good], w, None, torch.ones_like(x[good]), None)
    for out in (y, codes.float(), scales, dx):
        assert torch.isfinite(out[good]).all()
    assert not y[0].any() and not codes[0].float().any()
    assert y[4].isnan().all() and dx[4].isnan().all() and y[3, 3].isnan()


def test_empty_and_refusals(cuda_device):
    x, w = torch.randn(4, 8, device=cuda_device), torch.ones(8, device=cuda_device)
    y, total, rstd = ops.rms_norm(x[:0], w, x[:0])
    assert y.shape == total.shape == (0, 8)
    codes, scales, _, _ = ops.rms_norm_8bit(x[:0], w)
    assert codes.shape == (0, 8) and scales.shape == (0, 1)
    dx, dweight = ops.rms_norm_backward(x[:0], x[:0], w, rstd)
    assert dx.shape == (0, 8) and not dweight.any()
    y, total, rstd = ops.rms_norm(x, w)
    with pytest.raises(ValueError, match="residual"):
        ops.rms_norm(x, w, x[:2])
    with pytest.raises(TypeError, match="share"):
        ops.rms_norm_8bit(x, w, x.half())
    with pytest.raises(ValueError, match="last dimension"):
        ops.rms_norm(x, w[:4])
    with pytest.raises(ValueError, match="grad"):
        ops.rms_norm_backward(x[:2], total, w, rstd)
    with pytest.raises(ValueError, match="rstd"):
        ops.rms_norm_backward(x, total, w, rstd[:2])
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.rms_norm(x.double(), w)
