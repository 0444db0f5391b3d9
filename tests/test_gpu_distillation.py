"""The distillation loss and its gradient against the formula in 64 bits.

Bounds (u = 2^-24, ex2.approx off by at most 2^-22): an exponential of d = (z - m) / T errs by
2^-22 + 4 u |d| of itself (the difference is rounded, scaled and the scale is rounded); a sum of V of
them by those errors' mean under q and 64 + V / 4096 roundings. So log s errs by
e_s = 2^-22 + 4 u mean_q |d| + (64 + V / 4096) u, q_i by (2^-22 + 4 u |d_i| + e_s) q_i, the teacher's p
alike. The loss is a sum of terms p_j (log p_j - log q_j) whose logarithms err by their exponentials'
bounds and two roundings of their size each."""

from __future__ import annotations

import math

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops

pytestmark = pytest.mark.gpu

U, EX2 = 2.0**-24, 2.0**-22


def formula(logits, indices, teacher, temperature, grad):
    """(loss, its bound, dlogits, its bound), in 64 bits."""
    rows, v = logits.shape
    z, t = logits.double() / temperature, teacher.double() / temperature
    there = (indices >= 0) & (indices < v)
    t = torch.where(there, t, -math.inf)
    there = there & (t > -math.inf)
    some = there.any(1)
    top = torch.where(some, t.amax(1), 0.0)[:, None]
    d_t = torch.where(there, t - top, 0.0)
    p = torch.where(there, d_t.exp(), 0.0)
    total = torch.where(some, p.sum(1), 1.0)[:, None]
    p = p / total
    log_p = d_t - total.log()
    m = z.amax(1, keepdim=True)
    d = z - m
    s = d.exp().sum(1, keepdim=True)
    q = d.exp() / s
    at = torch.where(there, indices, 0).long()
    d_z = torch.where(there, d.gather(1, at), 0.0)
    log_q = d_z - s.log()
    size = torch.where(q > 0, d.abs(), 0.0)
    e_s = EX2 + 4 * U * (q * size).sum(1, keepdim=True) + (64 + v / 4096) * U
    e_p = 2 * EX2 + 8 * U * d_t.abs() + (64 + indices.shape[1]) * U
    t2 = temperature**2
    loss = t2 * torch.where(there, p * (log_p - log_q), 0.0).sum(1)
    term = log_p.abs() + log_q.abs()
    error = t2 * torch.where(there, p * (e_p * (1 + term) + e_s + 8 * U * (term + d_t.abs() + d_z.abs() + 1)), 0.0).sum(1)
    error = error + 64 * U * t2 * torch.where(there, p * term, 0.0).sum(1)
    g = torch.where(some, grad.double(), 0.0)[:, None] * temperature
    share = torch.zeros_like(z).scatter_add_(1, at, torch.where(there, p, 0.0))
    e_share = torch.zeros_like(z).scatter_add_(1, at, torch.where(there, p * e_p, 0.0))
    dz = torch.where(some[:, None], g * (q - share), 0.0)
    e_dz = torch.where(some[:, None], g.abs() * (q * (EX2 + 4 * U * size + e_s + 4 * U) + e_share + 4 * U * share), 0.0)
    return loss, error, dz, e_dz


def check(logits, indices, teacher, temperature=1.0, grad=None):
    rows = logits.shape[0]
    if grad is None:
        grad = torch.rand(rows, device=logits.device) + 0.5
    want, error, dz, e_dz = formula(logits, indices, teacher, temperature, grad)
    loss, statistics = ops.distillation_loss(logits, indices, teacher, temperature)
    both, dlogits = ops.distillation_loss_gradient(grad, logits, indices, teacher, temperature)
    apart = ops.distillation_loss_backward(grad, logits, indices, teacher, statistics, temperature)
    assert loss.shape == (rows,) and dlogits.shape == logits.shape and dlogits.dtype == logits.dtype
    # The calls share a row among different numbers of warps, so their sums differ in order.
    rounding = torch.finfo(logits.dtype).eps / 2
    bound = e_dz + rounding * (dz.abs() + e_dz) + (2.0**-25 if logits.dtype == torch.float16 else 1e-37)
    for values, gradient in ((loss, dlogits), (both, apart)):
        excess = ((values.double() - want).abs() - error).max().item()
        assert excess <= 0.0, f"loss: largest excess {excess}"
        excess = ((gradient.double() - dz).abs() - bound).max().item()
        assert excess <= 0.0, f"gradient: largest excess {excess}"
    return loss, dlogits


def inputs(device, rows, vocabulary, top, dtype, index_dtype=torch.int64, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    logits = (torch.randn(rows, vocabulary, generator=gen, device=device) * 3).to(dtype)
    indices = torch.randint(0, vocabulary, (rows, top), generator=gen, device=device)
    indices[torch.rand(rows, top, generator=gen, device=device) < 0.1] = -1
    teacher = torch.randn(rows, top, generator=gen, device=device) * 2 + 8
    return logits, indices.to(index_dtype), teacher


TYPES = (torch.bfloat16, torch.float16, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocabulary,top", [
    (1, 1, 1), (1, 2, 3), (3, 7, 2), (2, 31, 40), (5, 1000, 1), (1, 32000, 32), (7, 50001, 20), (40, 8192, 128),
    (400, 1025, 5), (600, 4099, 33), (9, 131072, 64), (3, 2049, 1024),
])
def test_loss(cuda_device, rows, vocabulary, top, dtype):
    """Indices come more than once where top is near the vocabulary's size."""
    for temperature, index_dtype in ((1.0, torch.int64), (2.5, torch.int32), (0.4, torch.int64)):
        logits, indices, teacher = inputs(cuda_device, rows, vocabulary, top, dtype, index_dtype)
        check(logits, indices, teacher.to(dtype) if temperature > 1 else teacher, temperature)


def test_rows_that_leave_nothing(cuda_device):
    logits, indices, teacher = inputs(cuda_device, 8, 5000, 6, torch.float32)
    indices[0] = -1
    indices[1] = 5000  # behind the vocabulary
    indices[2, 1:] = -7
    teacher[3] = -math.inf
    teacher[4, 2:] = -math.inf
    teacher[5] = torch.finfo(torch.float32).min
    logits[0], logits[1] = math.nan, -math.inf  # not read
    finite = torch.where(torch.isfinite(logits), logits, 0.0)
    grad = torch.rand(8, device=cuda_device) + 0.5
    loss, dlogits = ops.distillation_loss_gradient(grad, logits, indices, teacher, 2.0)
    check(finite, indices, teacher, 2.0, grad)
    want, want_dlogits = ops.distillation_loss_gradient(grad, finite, indices, teacher, 2.0)
    assert torch.equal(loss, want) and torch.equal(dlogits, want_dlogits)
    for r in (0, 1, 3):
        assert loss[r] == 0 and not dlogits[r].any()
    empty = ops.distillation_loss_gradient(grad, finite, indices[:, :0], teacher[:, :0])
    assert not empty[0].any() and not empty[1].any()


@pytest.mark.parametrize("rows", [4, 600])
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_vocabulary(cuda_device, dtype, rows):
    """Logits of -inf and of the type's lowest value have a share of zero, also a whole piece, and a
    thread's first pieces, of them; what is not finite stays in its row."""
    logits, indices, teacher = inputs(cuda_device, rows, 40000, 10, dtype)
    indices = indices.clamp_min(0) % 15000 + 20000
    logits[:, :20000] = -math.inf
    logits[:, 36000:] = torch.finfo(dtype).min
    check(logits, indices, teacher, 0.5)
    check(logits, indices, teacher, 1.0)
    broken = logits.clone()
    broken[1, 30000] = math.nan
    broken[2, 39999] = math.inf
    broken[3] = -math.inf
    grad = torch.ones(rows, device=cuda_device)
    loss, dlogits = ops.distillation_loss_gradient(grad, broken, indices, teacher)
    want, want_dlogits = ops.distillation_loss_gradient(grad, logits, indices, teacher)
    others = [0, *range(4, rows)]
    assert loss[1:4].isnan().all() and dlogits[1:4].isnan().all()
    assert torch.equal(loss[others], want[others]) and torch.equal(dlogits[others], want_dlogits[others])
    # A teacher's choice that the student rules out costs infinitely much; its gradient does not.
    logits[0, indices[0, 0]] = -math.inf
    loss, dlogits = ops.distillation_loss_gradient(grad, logits, indices, teacher)
    assert loss[0] == math.inf and torch.isfinite(dlogits).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_logits(cuda_device, dtype):
    """Differences count, not sizes: rows of 3e4 and rows of the lowest value alone."""
    logits, indices, teacher = inputs(cuda_device, 5, 3001, 8, dtype)
    logits = (logits.float() + 30000).to(dtype)
    logits[3] = torch.finfo(dtype).min
    check(logits, indices.clamp_min(0), teacher, 0.25)


@pytest.mark.parametrize("rows", [3, 500])
def test_views(cuda_device, rows):
    """Strided rows that start anywhere, turned indices, rows apart in the teacher's tensors."""
    for dtype in TYPES:
        wide, indices, teacher = inputs(cuda_device, 2 * rows, 3000, 9, dtype)
        check(wide[::2, 3:2504], (indices % 2501)[1::2], teacher[:rows])
        check(wide[:rows, 8:1009], (indices % 1001)[:rows].t().contiguous().t(), teacher[rows:].t().contiguous().t())


@pytest.mark.parametrize("vocabulary", [100, 70000])
def test_one_index_many_times(cuda_device, vocabulary):
    logits, _, teacher = inputs(cuda_device, 6, vocabulary, 1000, torch.float32)
    indices = torch.full((6, 1000), 57, device=cuda_device)
    indices[1::2, ::3] = 99
    check(logits, indices, teacher)


def test_refusals(cuda_device):
    logits, indices, teacher = inputs(cuda_device, 4, 100, 3, torch.float32)
    grad = torch.ones(4, device=cuda_device)
    _, statistics = ops.distillation_loss(logits, indices, teacher)
    with pytest.raises(ValueError, match="vocabulary"):
        ops.distillation_loss(logits[0], indices, teacher)
    with pytest.raises(ValueError, match="top"):
        ops.distillation_loss(logits, indices, teacher[:, :2])
    with pytest.raises(ValueError, match="top"):
        ops.distillation_loss(logits, indices[:3], teacher[:3])
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.distillation_loss(logits, indices.short(), teacher)
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.distillation_loss(logits.double(), indices, teacher)
    with pytest.raises(RuntimeError, match="temperature"):
        ops.distillation_loss(logits, indices, teacher, 0.0)
    with pytest.raises(RuntimeError, match="temperature"):
        ops.distillation_loss(logits, indices, teacher, math.nan)
    with pytest.raises(RuntimeError, match="1024"):
        ops.distillation_loss(logits, indices[:, :1].expand(4, 1025), teacher[:, :1].expand(4, 1025))
    with pytest.raises(ValueError, match="grad"):
        ops.distillation_loss_gradient(grad[:2], logits, indices, teacher)
    with pytest.raises(ValueError, match="grad"):
        ops.distillation_loss_backward(grad.half(), logits, indices, teacher, statistics)
    with pytest.raises(ValueError, match="statistics"):
        ops.distillation_loss_backward(grad, logits, indices, teacher, statistics[:2])
    loss, statistics = ops.distillation_loss(logits[:0], indices[:0], teacher[:0])
    assert loss.shape == (0,) and statistics.shape == (0, 2)
