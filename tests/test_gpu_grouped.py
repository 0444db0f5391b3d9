"""Products grouped by expert against 64-bit products of the same inputs.

Bound of an element: the fp32 sum of K products errs by at most K 2^-23 sum|a b|
(one rounding for each addition, a bit more than that if the adder truncates),
and the result is rounded once to the output type (half an epsilon of it, or half
of float16's smallest step, 2^-25)."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops

pytestmark = pytest.mark.gpu

ROUNDING = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}  # unit roundoff


def ends_of(counts, device, dtype=torch.int32):
    return torch.tensor(counts, device=device).cumsum(0).to(dtype)


def normal(gen, *shape, dtype, device, scale=1.0):
    return (torch.randn(shape, generator=gen, device=device) * scale).to(dtype)


def assert_close(out, exact, magnitude, terms):
    sums = terms * 2.0**-23 * magnitude
    bound = sums + ROUNDING[out.dtype] * (exact.abs() + sums) + 2.0**-25
    error = (out.double() - exact).abs()
    worst = (error - bound).max().item() if out.numel() else 0.0
    assert worst <= 0.0, f"off by {error.max().item()} (largest excess {worst})"


def by_group(left, right, counts):
    """Exact rows product and its magnitude, from 64-bit products group by group."""
    exact = torch.zeros((left.shape[0], right.shape[2]), dtype=torch.float64, device=left.device)
    magnitude = torch.zeros_like(exact)
    at = 0
    for e, n in enumerate(counts):
        a, b = left[at:at + n].double(), right[e].double()
        exact[at:at + n] = a @ b
        magnitude[at:at + n] = a.abs() @ b.abs()
        at += n
    return exact, magnitude


COUNTS = [
    [1],
    [0, 1, 0],
    [3, 0, 70, 1, 17],
    [0, 0, 0],
    [255, 256, 257, 0, 1],
    [600, 31, 33],
    [1] * 70,
    [0] * 40 + [90] + [0] * 30,
]


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("k,n", [(64, 128), (8, 8), (200, 264), (72, 1000)])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_product(cuda_device, counts, k, n, transposed, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    rows = sum(counts) + 5  # five rows that nobody owns
    left = normal(gen, rows, k, dtype=dtype, device=cuda_device)
    shape = (len(counts), n, k) if transposed else (len(counts), k, n)
    right = normal(gen, *shape, dtype=dtype, device=cuda_device, scale=0.1)
    if transposed:
        right = right.transpose(1, 2)
    out = ops.grouped_gemm(left, right, ends_of(counts, cuda_device))
    assert out.shape == (rows, n) and out.dtype == dtype
    exact, magnitude = by_group(left, right, counts)
    assert_close(out, exact, magnitude, k)
    assert not out[sum(counts):].any()


@pytest.mark.parametrize("k,n", [(1, 1), (7, 3), (65, 33), (1, 40), (40, 1), (129, 257)])
@pytest.mark.parametrize("transposed", [False, True])
def test_rows_product_odd_sizes(cuda_device, k, n, transposed):
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    counts = [5, 0, 200, 1]
    left = normal(gen, 206, k, dtype=torch.bfloat16, device=cuda_device)
    right = normal(gen, *((4, n, k) if transposed else (4, k, n)), dtype=torch.bfloat16, device=cuda_device)
    if transposed:
        right = right.transpose(1, 2)
    exact, magnitude = by_group(left, right, counts)
    assert_close(ops.grouped_gemm(left, right, ends_of(counts, cuda_device)), exact, magnitude, k)


@pytest.mark.parametrize("counts", [[1], [0, 5, 0, 33, 2], [64, 1, 40], [9] * 30, [100, 7]])
@pytest.mark.parametrize("k,n", [(520, 8), (1000, 328), (2048, 136), (8192, 512), (2051, 133)])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_rows_product_long_contractions(cuda_device, counts, k, n, transposed, out_dtype):
    """Few rows and a long contraction: tiles that several CTAs share."""
    gen = torch.Generator(device=cuda_device).manual_seed(17)
    rows = sum(counts) + 3
    left = normal(gen, rows, k, dtype=torch.bfloat16, device=cuda_device)
    shape = (len(counts), n, k) if transposed else (len(counts), k, n)
    right = normal(gen, *shape, dtype=torch.bfloat16, device=cuda_device, scale=0.1)
    if transposed:
        right = right.transpose(1, 2)
    left[sum(counts):] = float("nan")  # rows that nobody owns stay out
    runs = [ops.grouped_gemm(left, right, ends_of(counts, cuda_device), out_dtype=out_dtype) for _ in range(3)]
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
    left[sum(counts):] = 0
    exact, magnitude = by_group(left, right, counts)
    assert_close(runs[0], exact, magnitude, k)
    assert not runs[0][sum(counts):].any()


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("m,n", [(128, 64), (8, 8), (264, 200), (130, 520), (33, 7)])
@pytest.mark.parametrize("out_dtype", [None, torch.float32])
def test_reduced_product(cuda_device, counts, m, n, out_dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    rows = sum(counts) + 5
    left = normal(gen, rows, m, dtype=torch.bfloat16, device=cuda_device)
    right = normal(gen, rows, n, dtype=torch.bfloat16, device=cuda_device)
    out = ops.grouped_gemm_reduce(left, right, ends_of(counts, cuda_device), out_dtype)
    assert out.shape == (len(counts), m, n)
    at = 0
    for e, count in enumerate(counts):
        a, b = left[at:at + count].double(), right[at:at + count].double()
        assert_close(out[e], a.T @ b, a.abs().T @ b.abs(), max(count, 1))
        at += count


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_output_types(cuda_device, out_dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    for counts in ([40, 0, 7], [400, 300]):
        left = normal(gen, sum(counts), 128, dtype=torch.float16, device=cuda_device)
        right = normal(gen, len(counts), 128, 96, dtype=torch.float16, device=cuda_device, scale=0.1)
        out = ops.grouped_gemm(left, right, ends_of(counts, cuda_device, torch.int64), out_dtype)
        assert out.dtype == out_dtype
        exact, magnitude = by_group(left, right, counts)
        assert_close(out, exact, magnitude, 128)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("counts", [[30, 50, 16], [300, 290, 410]])
def test_other_groups_do_not_leak(cuda_device, bad, counts):
    """NaN or infinity in one group's rows, or in rows that nobody owns, stays there."""
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    rows = sum(counts) + 9
    left = normal(gen, rows, 192, dtype=torch.bfloat16, device=cuda_device)
    grad = normal(gen, rows, 136, dtype=torch.bfloat16, device=cuda_device)
    right = normal(gen, 3, 192, 136, dtype=torch.bfloat16, device=cuda_device)
    ends = ends_of(counts, cuda_device)
    clean_rows, clean_sums = ops.grouped_gemm(left, right, ends), ops.grouped_gemm_reduce(grad, left, ends)
    dirty = torch.zeros(rows, dtype=torch.bool, device=cuda_device)
    dirty[counts[0]:counts[0] + counts[1]] = True
    dirty[sum(counts):] = True
    left[dirty] = bad
    grad[dirty] = bad
    out = ops.grouped_gemm(left, right, ends)
    assert torch.equal(out[~dirty], clean_rows[~dirty])
    assert not out[sum(counts):].any()
    sums = ops.grouped_gemm_reduce(grad, left, ends)
    assert torch.equal(sums[[0, 2]], clean_sums[[0, 2]])
    assert not sums[1].isfinite().any()


def test_ends_are_clamped(cuda_device):
    """Ends that descend or leave the rows are read as the nearest sound ones."""
    gen = torch.Generator(device=cuda_device).manual_seed(6)
    left = normal(gen, 100, 64, dtype=torch.bfloat16, device=cuda_device)
    right = normal(gen, 5, 64, 64, dtype=torch.bfloat16, device=cuda_device)
    for dtype in (torch.int32, torch.int64):
        wild = torch.tensor([-5, 40, 20, 1 << 30, 60], device=cuda_device, dtype=dtype)
        sound = torch.tensor([0, 40, 40, 100, 100], device=cuda_device, dtype=dtype)
        assert torch.equal(ops.grouped_gemm(left, right, wild), ops.grouped_gemm(left, right, sound))
        assert torch.equal(ops.grouped_gemm_reduce(left, left, wild), ops.grouped_gemm_reduce(left, left, sound))


def test_strides(cuda_device):
    """Slices of wider buffers, misaligned bases and broadcast matrices."""
    gen = torch.Generator(device=cuda_device).manual_seed(7)
    counts = [33, 0, 90]
    ends = ends_of(counts, cuda_device)
    wide = normal(gen, 123, 200, dtype=torch.bfloat16, device=cuda_device)
    weights = normal(gen, 3, 150, 170, dtype=torch.bfloat16, device=cuda_device)
    for left in (wide[:, 8:104], wide[:, 3:99], wide[:, ::2][:, :96], wide.T.contiguous().T[:, :96]):
        for right in (weights[:, :96, 8:88], weights[:, 1:97, 5:85], weights[:1, :96, :80].expand(3, 96, 80)):
            exact, magnitude = by_group(left, right, counts)
            assert_close(ops.grouped_gemm(left, right, ends), exact, magnitude, 96)
        sums = ops.grouped_gemm_reduce(left, wide[:, 101:130], ends)
        assert torch.equal(sums, ops.grouped_gemm_reduce(left.contiguous(), wide[:, 101:130].contiguous(), ends))


def test_empty_sizes(cuda_device):
    left = torch.ones(4, 16, dtype=torch.bfloat16, device=cuda_device)
    ends = torch.tensor([2, 4], device=cuda_device)
    none = torch.empty(0, dtype=torch.int32, device=cuda_device)
    assert ops.grouped_gemm(left[:0], torch.ones_like(left)[:2, :, None].expand(2, 16, 8), ends * 0).shape == (0, 8)
    assert not ops.grouped_gemm(left, left.new_ones(0, 16, 8), none).any()
    assert not ops.grouped_gemm(left[:, :0], left.new_ones(2, 0, 8), ends).any()
    assert not ops.grouped_gemm_reduce(left[:0], left[:0], ends).any()
    assert ops.grouped_gemm_reduce(left, left, none).shape == (0, 16, 16)


def test_another_stream(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(8)
    counts = [100, 28]
    left = normal(gen, 128, 256, dtype=torch.bfloat16, device=cuda_device)
    right = normal(gen, 2, 256, 256, dtype=torch.bfloat16, device=cuda_device)
    ends = ends_of(counts, cuda_device)
    want = ops.grouped_gemm(left, right, ends), ops.grouped_gemm_reduce(left, left, ends)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.grouped_gemm(left, right, ends), ops.grouped_gemm_reduce(left, left, ends)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(cuda_device):
    left = torch.ones(4, 16, dtype=torch.bfloat16, device=cuda_device)
    right = torch.ones(2, 16, 8, dtype=torch.bfloat16, device=cuda_device)
    ends = torch.tensor([2, 4], device=cuda_device)
    with pytest.raises(TypeError, match="share dtype"):
        ops.grouped_gemm(left.float(), right.float(), ends)
    with pytest.raises(TypeError, match="share dtype"):
        ops.grouped_gemm(left.half(), right, ends)
    with pytest.raises(ValueError, match="incompatible shapes"):
        ops.grouped_gemm(left[:, :8], right, ends)
    with pytest.raises(ValueError, match="expected left"):
        ops.grouped_gemm(left, right[0], ends)
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.grouped_gemm(left, right, ends.float())
    with pytest.raises(ValueError, match="one row number"):
        ops.grouped_gemm(left, right, ends[:1])
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.grouped_gemm(left, right, ends.cpu())
    with pytest.raises(ValueError, match="rows"):
        ops.grouped_gemm_reduce(left, left[:3], ends)
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.grouped_gemm(left, right, ends, torch.float64)
    with pytest.raises(RuntimeError, match="1024 groups"):
        ops.grouped_gemm(left, right[:1].expand(1025, 16, 8), torch.zeros(1025, device=cuda_device, dtype=torch.int32))


@pytest.mark.parametrize("batch,rows,cols", [(1, 1, 1), (1, 3, 7), (2, 5, 8), (3, 17, 65), (1, 200, 1023), (4, 9, 16)])
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5, 7])
def test_rows_are_copied_as_they_are(cuda_device, batch, rows, cols, offset):
    """Slices that start on any element, with any row pitch, and transposed ones."""
    size = batch * rows * (cols + 3) + offset
    flat = torch.arange(size, device=cuda_device).to(torch.int16).view(torch.bfloat16)
    source = flat[offset:].view(batch, rows, cols + 3)[:, :, :cols]
    copy, place, pitch = ops._row_layout(source[-1])
    assert pitch % 8 == 0 and place % 16 == 0 or rows == 1
    assert torch.equal(ops.row_operand(source[-1]).view(torch.int16), source[-1].view(torch.int16))
    copy, place, *strides = ops._group_layout(source)
    assert torch.equal(copy.as_strided(source.shape, strides).contiguous().view(torch.int16),
                       source.contiguous().view(torch.int16))
    turned = source.transpose(1, 2)
    copy, place, *strides = ops._group_layout(turned)
    assert torch.equal(copy.as_strided(turned.shape, strides).contiguous().view(torch.int16),
                       turned.contiguous().view(torch.int16))
