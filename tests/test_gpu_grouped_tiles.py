"""Every kernel of the rows product, at sizes that the choice sends to it.

Bounds as in test_gpu_grouped.py: K 2^-23 sum|a b| for an fp32 sum of K products, and one
rounding to the output type."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops
from test_gpu_grouped import assert_close, ends_of, normal

# (rows of a tile, CTAs that share it), rows of the groups, k, n
CASES = [
    ((64, 1), [40, 0, 33, 5], 1000, 1000),
    ((64, 1), [0, 1, 0, 0, 1, 0, 1, 1] * 8, 1024, 4096),  # several turns
    ((64, 2), [3, 0, 7, 1] * 16, 4096, 1024),
    ((64, 4), [7, 0, 33, 64, 1, 0, 2, 30, 9, 5], 8192, 2048),
    ((64, 8), [3, 2], 8192, 512),
    ((128, 1), [130, 0, 1, 97, 40, 17, 31, 70], 2048, 2048),
    ((128, 1), [300, 250, 0, 199, 20], 1000, 1501),
    ((256, 1), [500, 3, 0, 1400, 90], 72, 1501),
    ((256, 1), [1, 4000, 256, 0, 257, 700, 3700], 136, 3001),  # six turns of the pairs
    ((256, 1), [600, 0, 1000, 255, 513, 31, 200, 1900, 33, 60, 3, 900, 80, 130, 250, 5, 20, 0, 9, 1], 264, 3000),
    ((512, 1), [5000, 513, 2687], 2056, 7168),
    ((512, 1), [4097, 4100], 2048, 7161),
]
TAIL = 40  # rows that nobody owns


def test_every_kernel_has_a_case():
    assert {kernel for kernel, *_ in CASES} == {(64, 1), (64, 2), (64, 4), (64, 8), (128, 1), (256, 1), (512, 1)}


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,counts,k,n", CASES)
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_rows_product(cuda_device, kernel, counts, k, n, transposed, out_dtype):
    """With NaN in one group's rows and in those that nobody owns, and other products between."""
    rows, groups = sum(counts) + TAIL, len(counts)
    assert ops.grouped_gemm_plan(rows, n, k, groups) == kernel
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    left = normal(gen, rows, k, dtype=torch.bfloat16, device=cuda_device)
    shape = (groups, n, k) if transposed else (groups, k, n)
    right = normal(gen, *shape, dtype=torch.bfloat16, device=cuda_device, scale=0.1)
    if transposed:
        right = right.transpose(1, 2)
    ends = ends_of(counts, cuda_device)
    dirty = max(e for e, c in enumerate(counts) if c > 0 and e < groups - 1)  # not the last group
    starts = [sum(counts[:e]) for e in range(groups)]
    left[starts[dirty]:starts[dirty] + counts[dirty]] = float("nan")
    left[sum(counts):] = float("nan")
    out = ops.grouped_gemm(left, right, ends, out_dtype)
    ops.grouped_gemm(left[:50, :64], right[:2, :64, :72], ends_of([20, 25], cuda_device))
    assert torch.equal(out.nan_to_num(7.0), ops.grouped_gemm(left, right, ends, out_dtype).nan_to_num(7.0))
    assert out.dtype == out_dtype and not out[sum(counts):].any()
    for e, count in enumerate(counts):
        mine = out[starts[e]:starts[e] + count]
        if e == dirty:
            assert mine.isnan().all()
            continue
        a, b = left[starts[e]:starts[e] + count].double(), right[e].double()
        assert_close(mine, a @ b, a.abs() @ b.abs(), k)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1000, 1001])
@pytest.mark.parametrize("owned", [0, 300, 19000])
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.float32])
def test_buffers_that_are_mostly_unowned(cuda_device, n, owned, out_dtype):
    """A buffer padded to a capacity: its unowned rows come out zero, whatever they hold."""
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    counts = [owned // 2, 0, owned - owned // 2]
    left = normal(gen, 20000, 136, dtype=torch.float16, device=cuda_device)
    right = normal(gen, 3, 136, n, dtype=torch.float16, device=cuda_device, scale=0.1)
    left[owned:] = float("inf")
    out = ops.grouped_gemm(left, right, ends_of(counts, cuda_device), out_dtype)
    assert not out[owned:].any()
    a = left[:owned].double()
    half = owned // 2
    exact = torch.cat([a[:half] @ right[0].double(), a[half:] @ right[2].double()])
    magnitude = torch.cat([a[:half].abs() @ right[0].double().abs(), a[half:].abs() @ right[2].double().abs()])
    assert_close(out[:owned], exact, magnitude, 136)
    sums = ops.grouped_gemm_reduce(left, left[:, :72], ends_of(counts, cuda_device), torch.float32)
    assert sums.isfinite().all() and not sums[1].any()
