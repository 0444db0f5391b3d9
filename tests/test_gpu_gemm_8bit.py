"""Products of 8-bit matrices with scales for blocks of 128, and the quantiser, against 64 bits.

Codes and scales are held to the formula's own fp32 operations, bit for bit. A product's bound: the
tensor cores add the 128 terms of a block in fp32, each addition off by at most 2^-23 of the terms'
magnitudes (they may truncate), a block's sum is scaled (the scales' product and the scaling round
once each) and added up in fp32, 2^-24 each; the result is rounded once to its type."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops

pytestmark = pytest.mark.gpu

BLOCK = 128
LEAST = 448.0 * 2.0**-126
TYPES = (torch.bfloat16, torch.float16, torch.float32)


def quantized(x, block_rows):
    """The formula with torch's fp32 operations: (codes, scales)."""
    rows, columns = x.shape
    tall = -(-rows // block_rows) * block_rows
    padded = torch.nn.functional.pad(x.float(), (0, -columns % BLOCK, 0, tall - rows))
    blocks = padded.view(tall // block_rows, block_rows, -1, BLOCK)
    top = torch.where(blocks.isnan(), 0.0, blocks.abs()).amax((1, 3)).clamp_min(LEAST)
    # A number over a tensor would be its reciprocal times the number, rounded twice.
    scaled = (blocks * (torch.full_like(top, 448.0) / top)[:, None, :, None]).clamp(-448, 448).reshape(tall, -1)[:rows, :columns]
    return scaled.to(torch.float8_e4m3fn), top / torch.full_like(top, 448.0)


def values(codes, scales, block_rows):
    spread = scales.double().repeat_interleave(block_rows, 0)[: codes.shape[0]]
    return codes.double() * spread.repeat_interleave(BLOCK, 1)[:, : codes.shape[1]]


def same(codes, want):
    got, want = codes.float(), want.float()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def check_product(left, left_scales, right, right_scales, dtype, lv, rv):
    out = ops.gemm_8bit(left, left_scales, right, right_scales, out_dtype=dtype)
    assert out.dtype == dtype and out.shape == (left.shape[0], right.shape[1])
    exact, terms = lv @ rv, lv.abs() @ rv.abs()
    blocks = -(-left.shape[1] // BLOCK)
    error = (2 * BLOCK + blocks + 8) * 2.0**-24 * terms
    bound = error + torch.finfo(dtype).eps / 2 * (exact.abs() + error) + (2.0**-25 if dtype == torch.float16 else 1e-37)
    excess = ((out.double() - exact).abs() - bound).max().item()
    assert excess <= 0.0, f"largest excess {excess}"
    return out


def product(device, m, k, n, dtype, turned, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    x = normal(m, k) * torch.exp(normal(m, 1))
    w = 0.05 * normal(*((k, n) if turned else (n, k)))
    xc, xs = ops.quantize_8bit(x)
    wc, ws = ops.quantize_8bit(w, BLOCK)
    xv, wv = values(xc, xs, 1), values(wc, ws, BLOCK)
    if turned:
        return check_product(xc, xs, wc, ws, dtype, xv, wv)
    return check_product(xc, xs, wc.t(), ws.t(), dtype, xv, wv.t())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block_rows", [1, BLOCK])
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 128), (3, 130), (128, 256), (129, 1000), (300, 77), (513, 2049)])
def test_quantize(cuda_device, rows, columns, block_rows, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(rows)
    x = torch.randn(rows, columns, generator=gen, device=cuda_device) * torch.exp(
        4 * torch.randn(rows, 1, generator=gen, device=cuda_device))
    x = x.to(dtype)
    codes, scales = ops.quantize_8bit(x, block_rows)
    want, want_scales = quantized(x, block_rows)
    assert codes.shape == x.shape and codes.stride(0) % 16 == 0
    same(codes, want)
    assert torch.equal(scales, want_scales)


@pytest.mark.parametrize("block_rows", [1, BLOCK])
def test_quantize_views_and_extremes(cuda_device, block_rows):
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    base = torch.randn(140, 400, generator=gen, device=cuda_device)
    base[0, :256] = 0.0
    base[1, 3] = float("nan")
    base[2] = 1e-42
    base[3] *= 1e37
    base[130:] = 0.0
    for x in (base, base[:, 1:300], base[:, 4:388], base.t(), base[::3], base[:1].expand(140, 400), base.half(),
              base.bfloat16()[:, 1:]):
        x = torch.where(x.isinf(), 60000.0, x) if x.dtype == torch.float16 else x
        codes, scales = ops.quantize_8bit(x, block_rows)
        want, want_scales = quantized(x, block_rows)
        same(codes, want)
        assert torch.equal(scales, want_scales)
    # What lies behind a row's last column, up to 16 bytes, is zeros; an empty matrix has no codes.
    codes, _ = ops.quantize_8bit(base[:, :300], block_rows)
    assert codes.stride(0) == 304 and not codes.as_strided((140, 304), (304, 1))[:, 300:].float().any()
    for shape in ((0, 5), (5, 0)):
        codes, scales = ops.quantize_8bit(base.new_zeros(shape), block_rows)
        assert codes.shape == shape and scales.numel() == 0


def test_infinity_makes_its_block_nan(cuda_device):
    x = torch.ones(2, 256, device=cuda_device)
    x[0, 5] = float("inf")
    codes, scales = ops.quantize_8bit(x)
    assert scales[0, 0].isinf() and codes[0, 5].float().isnan() and torch.isfinite(scales[:, 1]).all()
    w, ws = ops.quantize_8bit(torch.ones(16, 256, device=cuda_device), BLOCK)
    out = ops.gemm_8bit(codes, scales, w.t(), ws.t())
    assert out[0].isnan().all() and (out[1] == 256).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("m,k,n", [
    (1, 1, 1), (1, 128, 128), (1, 4096, 1000), (2, 130, 17), (16, 512, 256), (17, 300, 384), (33, 1024, 129),
    (64, 2048, 640), (65, 100, 40), (100, 1408, 2000), (128, 128, 2048), (129, 128, 128), (129, 1, 3), (256, 256, 256),
    (257, 1000, 300), (700, 640, 1501), (1500, 384, 1040),
])
def test_product(cuda_device, m, k, n, turned, dtype):
    product(cuda_device, m, k, n, dtype, turned)


@pytest.mark.parametrize("m", [1, 5, 40, 120, 2000])
def test_product_of_operands_anywhere(cuda_device, m):
    """Operands and scales with odd offsets, strides and orders give the same bits as aligned ones."""
    gen = torch.Generator(device=cuda_device).manual_seed(m)
    k, n = 333, 210
    x = torch.randn(m, k, generator=gen, device=cuda_device)
    w = torch.randn(n, k, generator=gen, device=cuda_device)
    xc, xs = ops.quantize_8bit(x)
    wc, ws = ops.quantize_8bit(w, BLOCK)
    want = ops.gemm_8bit(xc, xs, wc.t(), ws.t())
    tight = [c.view(torch.uint8).contiguous().view(torch.float8_e4m3fn) for c in (xc, wc)]
    assert tight[0].stride(0) in (k, 1) or m == 1
    assert torch.equal(ops.gemm_8bit(tight[0], xs.contiguous(), tight[1].t(), ws.contiguous().t()), want)
    turned = [c.view(torch.uint8).t().contiguous().view(torch.float8_e4m3fn) for c in (xc, wc)]
    assert torch.equal(ops.gemm_8bit(turned[0].t(), xs, turned[1], ws.t()), want)
    wide = torch.zeros(2 * m + 1, k + 40, dtype=torch.uint8, device=cuda_device)[1::2, 7:7 + k]
    wide.copy_(xc.view(torch.uint8))
    assert torch.equal(ops.gemm_8bit(wide.view(torch.float8_e4m3fn), xs, wc.t(), ws.t()), want)


@pytest.mark.parametrize("m,k,n", [(5, 1, 7), (1, 1, 1), (200, 1, 1), (1, 20, 1), (40, 3, 1), (300, 16, 300)])
def test_product_of_thin_operands(cuda_device, m, k, n):
    """Without padding between rows, by rows and by columns: sizes of one leave strides undetermined."""
    x = torch.randn(m, k, device=cuda_device)
    w = torch.randn(n, k, device=cuda_device)
    xc, xs = ops.quantize_8bit(x)
    wc, ws = ops.quantize_8bit(w, BLOCK)
    want = ops.gemm_8bit(xc, xs, wc.t(), ws.t(), out_dtype=torch.float32)
    left, right = (c.view(torch.uint8).contiguous() for c in (xc, wc))
    f8 = torch.float8_e4m3fn
    for a in (left, left.t().contiguous().t()):
        for b in (right.t(), right.t().contiguous()):
            assert torch.equal(ops.gemm_8bit(a.view(f8), xs, b.view(f8), ws.t(), out_dtype=torch.float32), want)


def test_same_bits_on_every_run(cuda_device):
    for m, k, n in ((1, 4096, 512), (50, 4096, 256), (300, 1024, 600)):
        outs = [product(cuda_device, m, k, n, torch.float32, False, seed=7) for _ in range(3)]
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_nan_code_stays_in_its_row(cuda_device):
    """A NaN in the last, partial block reaches its own row only, and nothing behind the matrix enters."""
    for m in (3, 200):
        x = torch.randn(m, 200, device=cuda_device)
        x[1, 199] = float("nan")
        w = torch.randn(150, 200, device=cuda_device)
        out = ops.gemm_8bit(*ops.quantize_8bit(x), *(t.t() for t in ops.quantize_8bit(w, BLOCK)))
        assert out[1].isnan().all() and torch.isfinite(out[[0, *range(2, m)]]).all()


def test_refusals(cuda_device):
    x = torch.randn(4, 256, device=cuda_device)
    w = torch.randn(8, 256, device=cuda_device)
    xc, xs = ops.quantize_8bit(x)
    wc, ws = (t.t() for t in ops.quantize_8bit(w, BLOCK))
    with pytest.raises(ValueError, match="1 or 128"):
        ops.quantize_8bit(x, 64)
    with pytest.raises(ValueError, match="matrix"):
        ops.quantize_8bit(x[0])
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.quantize_8bit(x.double())
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops.gemm_8bit(x, xs, wc, ws)
    with pytest.raises(ValueError, match="incompatible"):
        ops.gemm_8bit(xc, xs, wc.t(), ws)
    with pytest.raises(ValueError, match="left_scales"):
        ops.gemm_8bit(xc, xs[:, :1], wc, ws)
    with pytest.raises(ValueError, match="right_scales"):
        ops.gemm_8bit(xc, xs, wc, ws[:1])
    with pytest.raises(TypeError, match="float32"):
        ops.gemm_8bit(xc, xs.half(), wc, ws)
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.gemm_8bit(xc, xs, wc, ws, out_dtype=torch.float64)
    empty = ops.gemm_8bit(xc[:, :0], xs[:, :0], wc[:0], ws[:0])
    assert empty.shape == (4, 8) and not empty.any()
    assert ops.gemm_8bit(xc[:0], xs[:0], wc, ws).shape == (0, 8)
