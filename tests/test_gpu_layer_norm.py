"""Layer norm forward and backward against the formulas in 64 bits.

Bounds: a sum over a row takes at most 64 roundings on any path (each thread's share,
then a tree), so the mean errs by 64 u mean|x| (u = 2^-24), a centred and scaled value h by
e_h = 64 u (|h| + r mean|x|); a sum over R rows by R u times the sum of magnitudes. Results
are rounded once to their type."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops

pytestmark = pytest.mark.gpu

ROUNDING = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}  # unit roundoff
U = 64 * 2.0**-24


def check(out, exact, error):
    absolute = 2.0**-25 if out.dtype == torch.float16 else 1e-40
    bound = error + ROUNDING[out.dtype] * (exact.abs() + error) + absolute
    worst = ((out.double() - exact).abs() - bound).max().item() if out.numel() else 0.0
    assert worst <= 0.0, f"largest excess {worst}"


def check_norm(x, weight, bias, grad, epsilon=1e-5):
    y, mean, rstd = ops.layer_norm(x, weight, bias, epsilon)
    columns = weight.numel()
    x64 = x.double().reshape(-1, columns)
    w64 = weight.double()
    b64 = bias.double() if bias is not None else torch.zeros_like(w64)
    mu = x64.mean(1, keepdim=True)
    r = 1 / (x64.sub(mu).square().mean(1, keepdim=True) + epsilon).sqrt()
    h = (x64 - mu) * r
    size = x64.abs().mean(1, keepdim=True)
    e_h = U * (h.abs() + r * size)
    check(mean.reshape(-1, 1), mu, U * size)
    check(rstd.reshape(-1, 1), r, U * r * (1 + r * size))
    check(y.reshape(-1, columns), h * w64 + b64, w64.abs() * e_h + U * ((h * w64).abs() + b64.abs()))
    if grad is None:
        return
    dx, dweight, dbias = ops.layer_norm_backward(grad, x, weight, mean, rstd)
    assert dx.shape == x.shape and dx.dtype == x.dtype and dweight.dtype == weight.dtype
    dy = grad.double().reshape(-1, columns)
    a = dy * w64
    c1, c2 = (a * h).mean(1, keepdim=True), a.mean(1, keepdim=True)
    s1, s2 = (a * h).abs().mean(1, keepdim=True), a.abs().mean(1, keepdim=True)
    e_1 = U * s1 + (a.abs() * e_h).mean(1, keepdim=True)
    want = r * (a - c2 - h * c1)
    error = r * (U * (a.abs() + s2) + h.abs() * e_1 + e_h * s1 + U * h.abs() * s1)
    check(dx.reshape(-1, columns), want, error + U * (1 + r * size) * want.abs())
    rows = max(x64.shape[0], 1)
    check(dweight, (dy * h).sum(0), (dy.abs() * e_h).sum(0) + rows * 2.0**-24 * (dy * h).abs().sum(0))
    check(dbias, dy.sum(0), rows * 2.0**-24 * dy.abs().sum(0))


def inputs(gen, rows, columns, dtype, w_dtype, device):
    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    x = (normal(rows, columns) * (0.5 + torch.rand((rows, 1), generator=gen, device=device)) + 0.3).to(dtype)
    return x, (1 + 0.2 * normal(columns)).to(w_dtype), normal(columns).to(w_dtype), normal(rows, columns).to(dtype)


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
         (torch.float32, torch.float32), (torch.float32, torch.bfloat16)]


@pytest.mark.parametrize("rows", [1, 5, 700])
@pytest.mark.parametrize("columns", [1, 2, 7, 64, 500, 512, 520, 1111, 2048, 4104, 8192, 9001])
@pytest.mark.parametrize("dtype,w_dtype", TYPES)
def test_norm(cuda_device, rows, columns, dtype, w_dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    x, weight, bias, grad = inputs(gen, rows, columns, dtype, w_dtype, cuda_device)
    check_norm(x, weight, bias, grad)


@pytest.mark.parametrize("rows,columns", [(3, 16384), (3, 16385), (200, 16376), (70, 20000), (2, 40001), (4000, 96)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_wide_and_long(cuda_device, rows, columns, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    x, weight, bias, grad = inputs(gen, rows, columns, dtype, torch.float32, cuda_device)
    check_norm(x, weight, bias, grad)


def test_shapes_strides_and_no_bias(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    x, weight, bias, grad = inputs(gen, 60, 264, torch.bfloat16, torch.bfloat16, cuda_device)
    check_norm(x.view(3, 4, 5, 264), weight, None, grad.view(3, 4, 5, 264))
    check_norm(x[:, :256], weight[:256], bias[:256], grad[:, 8:])
    check_norm(x[:, 1:258], weight[1:258], bias[1:258], grad[:, 3:260])
    check_norm(x[::2], weight, bias, grad[::2])
    check_norm(x.T.contiguous().T, weight, bias, grad)
    check_norm(x[:1].expand(60, 264), weight, bias, grad[:1].expand(60, 264))
    check_norm(x.view(3, 20, 264).transpose(0, 1), weight, bias, grad.view(20, 3, 264))
    check_norm(x[0], weight, bias, grad[0])


@pytest.mark.parametrize("rows", [2, 1500])
@pytest.mark.parametrize("columns", [513, 1024, 1027, 2053, 5003, 8200, 16381])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_that_start_anywhere(cuda_device, rows, columns, dtype):
    """Rows of x and of its gradient at different offsets, between rows of NaN."""
    gen = torch.Generator(device=cuda_device).manual_seed(7)
    values, weight, bias, grads = inputs(gen, rows, columns, dtype, torch.float32, cuda_device)
    nan = float("nan")
    wide = torch.full((rows + 2, columns + 6), nan, dtype=dtype, device=cuda_device)
    grad = torch.full((rows + 2, columns + 11), nan, dtype=dtype, device=cuda_device)
    x, dy = wide[1:-1, 1:columns + 1], grad[1:-1, 3:columns + 3]
    x.copy_(values)
    dy.copy_(grads)
    check_norm(x, weight, bias, dy)


def test_constant_and_large_rows(cuda_device):
    """Rows of one value (variance zero), rows far from zero, rows of large values."""
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    x, weight, bias, grad = inputs(gen, 8, 1000, torch.float32, torch.float32, cuda_device)
    x[1] = 3.0
    x[2] = 0.0
    x[3] += 1000.0
    x[4] *= 1e15
    x[5] *= 1e-15
    check_norm(x, weight, bias, grad)


def test_nonfinite_rows_stay_alone(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    x, weight, bias, grad = inputs(gen, 9, 520, torch.bfloat16, torch.float32, cuda_device)
    clean = ops.layer_norm(x, weight, bias, 1e-5)
    dx = ops.layer_norm_backward(grad, x, weight, *clean[1:])[0]
    x[4, 3] = float("nan")
    x[6, 5] = float("inf")
    keep = [0, 1, 2, 3, 5, 7, 8]
    y, mean, rstd = ops.layer_norm(x, weight, bias, 1e-5)
    assert torch.equal(y[keep], clean[0][keep]) and y[4].isnan().all() and not y[6].isfinite().all()
    assert torch.equal(ops.layer_norm_backward(grad, x, weight, mean, rstd)[0][keep], dx[keep])


def test_no_rows(cuda_device):
    x = torch.empty(0, 64, device=cuda_device)
    w = torch.ones(64, device=cuda_device)
    y, mean, rstd = ops.layer_norm(x, w, w, 1e-5)
    dx, dw, db = ops.layer_norm_backward(x, x, w, mean, rstd)
    assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()


def test_repeats_bit_for_bit(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(6)
    x, weight, _, grad = inputs(gen, 3001, 1024, torch.bfloat16, torch.float32, cuda_device)
    _, mean, rstd = ops.layer_norm(x, weight, None, 1e-5)
    first = ops.layer_norm_backward(grad, x, weight, mean, rstd)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = ops.layer_norm_backward(grad, x, weight, mean, rstd)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_refusals(cuda_device):
    x, w = torch.ones(4, 8, device=cuda_device), torch.ones(8, device=cuda_device)
    with pytest.raises(ValueError, match="last dimension"):
        ops.layer_norm(x, w[:4], None, 1e-5)
    with pytest.raises(ValueError, match="last dimension"):
        ops.layer_norm(x[:, :0], w[:0], None, 1e-5)
    with pytest.raises(ValueError, match="shapes differ"):
        ops.layer_norm(x, w, w[:4], 1e-5)
    with pytest.raises(TypeError, match="share a dtype"):
        ops.layer_norm(x, w, w.half(), 1e-5)
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.layer_norm(x.double(), w, None, 1e-5)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.layer_norm(x.cpu(), w.cpu(), None, 1e-5)
    y, mean, rstd = ops.layer_norm(x, w, None, 1e-5)
    with pytest.raises(ValueError, match="shapes differ"):
        ops.layer_norm_backward(y[:2], x, w, mean, rstd)
    with pytest.raises(TypeError, match="share a dtype"):
        ops.layer_norm_backward(y.half(), x, w, mean, rstd)
    with pytest.raises(ValueError, match="one entry per row"):
        ops.layer_norm_backward(y, x, w, mean[:2], rstd)
