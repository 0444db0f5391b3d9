"""Every kernel of the 8-bit product, at sizes that the choice sends to it, against 64 bits.

Bounds as in test_gpu_gemm_8bit.py: the tensor cores' fp32 additions within a block of 128, a
scaling and an addition a block (and a part), one rounding to the output's type."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops
from gram_newton_schulz_ampere_b200.training import linear_8bit
from test_gpu_gemm_8bit import BLOCK, TYPES, check_product, values

# (rows of a tile, CTAs that share it), m, k, n. Rings hold 4 to 6 blocks; where it says so, a CTA
# has more of them, and a pair more than one tile.
CASES = [
    ((16, 1), 9, 1000, 20001),  # 8 blocks a CTA
    ((16, 2), 2, 2000, 12801),
    ((16, 4), 16, 5000, 6400),  # 10
    ((16, 8), 1, 14336, 520),  # 14
    ((32, 1), 32, 2500, 40000),  # 20
    ((32, 2), 17, 2000, 12801),
    ((32, 4), 31, 5000, 6400),
    ((32, 8), 20, 8192, 300),  # 8
    ((128, 1), 1100, 2000, 1501),  # 16
    ((128, 2), 250, 2000, 4001),  # 8
    ((128, 4), 50, 4096, 256),  # 8
    ((128, 4), 100, 4100, 1501),  # 9, 8, 8 and 8
    ((256, 1), 2049, 1000, 1501),  # 8 blocks, rows of the output off 16 bytes
    ((256, 1), 5000, 1000, 1501),  # 120 tiles
    ((256, 1), 2500, 900, 1040),  # rows on 16 bytes, remainders of tiles both ways
    ((256, 1), 4097, 1500, 2000),  # 136 tiles of 12 blocks
    ((256, 1), 4600, 130, 1040),  # two blocks
    ((256, 1), 4600, 100, 1037),  # one
]


def factors(device, m, k, n, turned):
    """x [m, k] and w ([k, n] turned, else [n, k]) whose scales differ from row to row and from block to block."""
    gen = torch.Generator(device=device).manual_seed(11)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    def blocks(*shape):  # a power of two for each block of 128
        size = [-(-s // BLOCK) if s > 1 else 1 for s in shape]
        power = torch.exp2(torch.randint(-3, 4, size, generator=gen, device=device).float())
        for i, s in enumerate(shape):
            if s > 1:
                power = power.repeat_interleave(BLOCK, i).narrow(i, 0, s)
        return power

    x = normal(m, k) * torch.exp(normal(m, 1)) * blocks(1, k)
    shape = (k, n) if turned else (n, k)
    return x, 0.05 * normal(*shape) * blocks(*shape)


def test_every_kernel_has_a_case():
    assert {kernel for kernel, *_ in CASES} == {(rows, parts) for rows in (16, 32) for parts in (1, 2, 4, 8)} | {
        (128, 1), (128, 2), (128, 4), (256, 1)}


def test_plan_refusals(native_lib):
    tile, parts = ctypes.c_int(), ctypes.c_int()
    for arguments, words in (((-1, 1, 1), b"negative"), ((4, 1 << 23, 128), b"limits"), ((0, 4, 4), b"no plan"), ((4, 4, 0), b"no plan")):
        assert native_lib.gns_gemm_8bit_plan(*arguments, ctypes.byref(tile), ctypes.byref(parts)) < 0
        assert words in native_lib.gns_last_error()
    assert native_lib.gns_gemm_8bit_plan(4, 4, 4, None, ctypes.byref(parts)) < 0
    assert b"null" in native_lib.gns_last_error()


@pytest.mark.parametrize("kernel,m,k,n", CASES)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.gpu
def test_product(cuda_device, kernel, m, k, n, turned, dtype):
    """Right stored by columns and by rows, each type of output; the same bits again behind another product."""
    assert ops.gemm_8bit_plan(m, n, k) == kernel
    x, w = factors(cuda_device, m, k, n, turned)
    xc, xs = ops.quantize_8bit(x)
    wc, ws = ops.quantize_8bit(w, BLOCK)
    xv, wv = values(xc, xs, 1), values(wc, ws, BLOCK)
    right = (wc, ws) if turned else (wc.t(), ws.t())
    out = check_product(xc, xs, *right, dtype, xv, wv if turned else wv.t())
    ops.gemm_8bit(xc[:5], xs[:5], *right)
    assert torch.equal(out, ops.gemm_8bit(xc, xs, *right, out_dtype=dtype))


@pytest.mark.parametrize("kernel,m,k,n", [c for c in CASES if c[2] % BLOCK > 1])
@pytest.mark.gpu
def test_nan_stays_in_its_row_and_column(cuda_device, kernel, m, k, n):
    """Codes of NaN in the last, partial block reach a row and a column, and nothing behind the matrices enters."""
    assert ops.gemm_8bit_plan(m, n, k) == kernel
    x, w = factors(cuda_device, m, k, n, False)
    clean = ops.gemm_8bit(*ops.quantize_8bit(x), *(t.t() for t in ops.quantize_8bit(w, BLOCK)))
    assert torch.isfinite(clean).all()
    x[m - 1, k - 1] = float("nan")
    w[n - 1, k - 1] = float("nan")
    out = ops.gemm_8bit(*ops.quantize_8bit(x), *(t.t() for t in ops.quantize_8bit(w, BLOCK)))
    assert out[m - 1].isnan().all() and out[:, n - 1].isnan().all()
    # The scales of their blocks do not see a NaN; those of the values beside them may have grown less.
    assert torch.isfinite(out[: m - 1, : n - 1]).all()
    far = (n - 1) // BLOCK * BLOCK
    assert torch.equal(out[: m - 1, :far], clean[: m - 1, :far])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,n", [(2500, 1040, 1501), (5000, 1501, 1040)])
def test_linear_layer_of_many_rows(cuda_device, rows, k, n, dtype):
    """Output and input gradient both take the kernel for many rows, one operand by columns, one by rows."""
    assert ops.gemm_8bit_plan(rows, n, k) == ops.gemm_8bit_plan(rows, k, n) == (256, 1)
    gen = torch.Generator(device=cuda_device).manual_seed(12)
    x, w, dy = (torch.randn(shape, generator=gen, device=cuda_device).to(dtype) for shape in ((rows, k), (n, k), (rows, n)))
    x.requires_grad_()
    w = (0.1 * w).requires_grad_()
    y = linear_8bit(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    codes, scales = ops.quantize_8bit(w.detach(), BLOCK)
    wv = values(codes, scales, BLOCK)
    for got, left, right in ((y, x.detach(), (codes.t(), scales.t(), wv.t())), (dx, dy, (codes, scales, wv))):
        lc, ls = ops.quantize_8bit(left)
        assert torch.equal(got, check_product(lc, ls, *right[:2], dtype, values(lc, ls, 1), right[2]))
    assert torch.equal(dw, ops.gemm(ops.row_operand(dy).t(), ops.row_operand(x.detach())))
