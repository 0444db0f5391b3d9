"""The distillation loss where a CTA has several rows, with rows between them that leave nothing, in every
kernel that the choice has: by a row's length, and by the bytes of rows under way.

Sizes follow from the number of SMs: CTAs of four warps (rows of up to 64 KB), eight an SM; of
sixteen, two an SM; and, for the loss with its gradient and rows of more than 160 KB, of
thirty-two, one an SM. Where more than 48 MB of rows are under way, what the second pass has read
leaves L2 first."""

from __future__ import annotations

import math

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops
from test_gpu_distillation import check, inputs

pytestmark = pytest.mark.gpu

KB, UNDER_WAY = 1024, 48 * 1024 * 1024

# warps of a CTA (loss and gradient in one call), rows a CTA, second pass's reads leave L2 first,
# vocabulary, type
CASES = [
    (4, 2.6, False, 4099, torch.float32),  # 8 or 9 slots of 2 KB for three warps
    (4, 2.2, False, 1025, torch.bfloat16),  # one or two: warps without any
    (4, 3.1, False, 300, torch.float16),
    (4, 1.1, True, 16001, torch.float32),
    (16, 2.4, False, 40000, torch.bfloat16),
    (16, 2.3, False, 40001, torch.float32),
    (32, 2.8, False, 100003, torch.bfloat16),
    (32, 2.7, True, 100003, torch.float32),
    (32, 3.2, True, 180000, torch.float16),
]


def rows_of(device, warps, share, vocabulary, dtype, leaves):
    """A number of rows, having checked that the case is what it says."""
    sms = torch.cuda.get_device_properties(device).multi_processor_count
    ctas = 32 // warps * sms
    rows = int(share * ctas)
    row = vocabulary * torch.empty((), dtype=dtype).element_size()
    assert rows > ctas and warps == (4 if row <= 64 * KB else 32 if row > 160 * KB else 16)
    assert (ctas * row > UNDER_WAY) == leaves
    return rows, ctas


@pytest.mark.parametrize("warps,share,leaves,vocabulary,dtype", CASES)
@pytest.mark.parametrize("empty", ["none", "some", "most"])
def test_several_rows_of_a_cta(cuda_device, warps, share, leaves, vocabulary, dtype, empty):
    """Loss, gradient from statistics and both in one call, against the formula; the rows that have no
    entries hold NaN and infinities. The first and the last row, rows that follow one another in a
    CTA, and all rows of one CTA are among them."""
    rows, ctas = rows_of(cuda_device, warps, share, vocabulary, dtype, leaves)
    logits, indices, teacher = inputs(cuda_device, rows, vocabulary, 5, dtype, seed=rows)
    gen = torch.Generator(device=cuda_device).manual_seed(rows)
    out = torch.rand(rows, generator=gen, device=cuda_device) < {"none": -1.0, "some": 0.35, "most": 0.9}[empty]
    if empty != "none":
        out[0] = out[-1] = True
        out[3::ctas] = True
        out[7], out[7 + ctas if 7 + ctas < rows else 7] = False, True
    indices[out, :] = -1
    indices[~out, 0] = indices[~out, 0].clamp_min(0)  # the others have an entry
    logits[out] = math.nan
    logits[out, ::7] = math.inf
    grad = torch.rand(rows, generator=gen, device=cuda_device) + 0.5
    grad[out] = math.nan
    loss, dlogits = check(logits, indices, teacher, 2.0, grad)
    assert not loss[out].any() and not dlogits[out].any()


@pytest.mark.parametrize("warps,share,leaves,vocabulary,dtype", CASES)
def test_few_rows_give_the_same(cuda_device, warps, share, leaves, vocabulary, dtype):
    """As many rows as CTAs, one each: the same bits as among several rows a CTA. The rows stay where they
    are: how many elements come before a multiple of 16 bytes decides which warp adds which."""
    rows, ctas = rows_of(cuda_device, warps, share, vocabulary, dtype, leaves)
    logits, indices, teacher = inputs(cuda_device, rows, vocabulary, 9, dtype, torch.int32, seed=1)
    indices[::4] = -1
    grad = torch.rand(rows, device=cuda_device)
    loss, dlogits = ops.distillation_loss_gradient(grad, logits, indices, teacher)
    for part in (slice(0, ctas), slice(rows - ctas, rows)):
        want, want_dlogits = ops.distillation_loss_gradient(grad[part], logits[part], indices[part], teacher[part])
        assert torch.equal(loss[part], want) and torch.equal(dlogits[part], want_dlogits)


def test_many_entries(cuda_device):
    """1024 entries a row: their lists leave room for fewer CTAs on an SM than there are of them."""
    for rows, vocabulary, dtype in ((1300, 4001, torch.bfloat16), (400, 90001, torch.float32)):
        logits, indices, teacher = inputs(cuda_device, rows, vocabulary, 1024, dtype, seed=2)
        indices[::3] = -1
        check(logits, indices, teacher, 0.8)
