"""The differentiable norm, 8-bit linear layers and distillation loss, and a run of them together."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

from gram_newton_schulz_ampere_b200 import Muon, ops
from gram_newton_schulz_ampere_b200.training import distillation_loss, linear_8bit, rms_norm, rms_norm_linear_8bit

pytestmark = pytest.mark.gpu

BLOCK = 128


def values(x, block_rows):
    """A matrix as its codes and scales hold it, in 64 bits."""
    codes, scales = ops.quantize_8bit(x, block_rows)
    spread = scales.double().repeat_interleave(block_rows, 0)[: x.shape[0]]
    return codes.double() * spread.repeat_interleave(BLOCK, 1)[:, : x.shape[1]]


def close(got, want, terms, count):
    """One rounding to the result's type (which is at most half a step) and sums of `count` products in
    fp32 whose additions may truncate: 2^-23 each of the terms' magnitudes."""
    error = (count + 300) * 2.0**-23 * terms
    bound = error + torch.finfo(got.dtype).eps / 2 * (want.abs() + error) + 2.0**-25
    assert ((got.double() - want).abs() <= bound).all()


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=gen.device)


@pytest.fixture
def gen(cuda_device):
    return torch.Generator(device=cuda_device).manual_seed(5)


def test_rms_norm_gradient_against_differences(gen):
    """Central differences of the fp32 operator along random directions. With steps of 2^-7 the
    third-order term and the rounding of a sum of 600 terms of size one are both near 1e-3 of
    the sum of magnitudes; the bound is 1e-2 of it."""
    inputs = [normal(gen, 6, 100), 1 + 0.1 * normal(gen, 100), normal(gen, 6, 100)]
    dy, dt = normal(gen, 6, 100), normal(gen, 6, 100)
    leaves = [t.clone().requires_grad_() for t in inputs]
    torch.autograd.backward(rms_norm(*leaves), (dy, dt))
    for i, leaf in enumerate(leaves):
        direction, step = normal(gen, *leaf.shape), 2.0**-7

        def value(sign):
            moved = [t + sign * step * direction if j == i else t for j, t in enumerate(inputs)]
            y, total = rms_norm(*moved)
            return (y.double() * dy.double()).sum() + (total.double() * dt.double()).sum()

        slope = (value(1) - value(-1)) / (2 * step)
        products = leaf.grad.double() * direction.double()
        assert abs((slope - products.sum()).item()) <= 1e-2 * products.abs().sum().item()


def test_rms_norm_uses(gen):
    """Only the norm, only the stream, or neither of the inputs needs a gradient."""
    x, r = (normal(gen, 3, 5, 64).bfloat16().requires_grad_() for _ in range(2))
    w = torch.ones(64, device=gen.device, requires_grad=True)
    y, total = rms_norm(x, w, r)
    assert y.shape == total.shape == x.shape
    gx, gr = torch.autograd.grad(total.sum(), (x, r), retain_graph=True)
    assert (gx == 1).all() and (gr == 1).all()
    assert torch.autograd.grad(total.sum(), w, allow_unused=True, retain_graph=True)[0] is None
    both = torch.autograd.grad(y.float().square().sum(), (x, w, r))
    assert torch.equal(both[0], both[2])
    alone = rms_norm(x, w)
    assert isinstance(alone, torch.Tensor) and torch.equal(alone, ops.rms_norm(x, w)[0])
    assert not rms_norm(x.detach(), w.detach()).requires_grad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,n", [(1, 128, 64), (20, 200, 333), (260, 640, 512)])
def test_linear_8bit(gen, rows, k, n, dtype):
    """Forward and the input's gradient are products of what 8 bits hold; the weight's of the factors themselves."""
    x = normal(gen, 2, rows, k).to(dtype).requires_grad_()
    w = (0.1 * normal(gen, n, k)).to(dtype).requires_grad_()
    dy = (0.1 * normal(gen, 2, rows, n)).to(dtype)
    y = linear_8bit(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.shape == (2, rows, n) and dx.shape == x.shape and dw.dtype == dtype
    flat, grad = x.detach().reshape(-1, k), dy.reshape(-1, n)
    x8, w8, g8 = values(flat, 1), values(w.detach(), BLOCK), values(grad, 1)
    close(y.detach().reshape(-1, n), x8 @ w8.T, x8.abs() @ w8.abs().T, k)
    close(dx.reshape(-1, k), g8 @ w8, g8.abs() @ w8.abs(), n)
    close(dw, grad.double().T @ flat.double(), grad.double().abs().T @ flat.double().abs(), 2 * rows)


def test_linear_8bit_views_and_frozen_factors(gen):
    x = normal(gen, 300, 150).bfloat16().t()[:, ::2].requires_grad_()  # [150, 150], strided
    w = normal(gen, 70, 150).bfloat16()
    y = linear_8bit(x, w)
    y.sum().backward()  # an expanded gradient
    want = linear_8bit(x.detach().contiguous().requires_grad_(), w)
    assert torch.equal(y, want) and x.grad.shape == x.shape and w.grad is None
    w.requires_grad_()
    linear_8bit(x.detach(), w).sum().backward()
    assert w.grad is not None
    empty = linear_8bit(x.detach()[:0], w)
    empty.sum().backward()
    assert empty.shape == (0, 70)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (1, 5, 130), (37, 129, 1), (300, 1, 70), (65, 257, 131), (129, 512, 384)])
def test_linear_8bit_is_its_parts(gen, rows, k, n, dtype):
    """The layer makes the calls that a user may make one by one: the same bits."""
    x = normal(gen, rows, k).to(dtype).requires_grad_()
    w = normal(gen, n, k).to(dtype).requires_grad_()
    dy = normal(gen, rows, n).to(dtype)
    y = linear_8bit(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    codes, scales = ops.quantize_8bit(w.detach(), BLOCK)
    assert torch.equal(y, ops.gemm_8bit(*ops.quantize_8bit(x.detach()), codes.t(), scales.t(), out_dtype=dtype))
    assert torch.equal(dx, ops.gemm_8bit(*ops.quantize_8bit(dy), codes, scales, out_dtype=dtype))
    assert torch.equal(dw, ops.gemm(ops.row_operand(dy).t(), ops.row_operand(x.detach())))


def test_linear_8bit_rows_that_start_anywhere(gen):
    """One row with an odd stride, rows from an odd address, a weight's columns out of a wider matrix."""
    wide = normal(gen, 9, 141).bfloat16()
    w = normal(gen, 50, 300).bfloat16()[:, 7:136].requires_grad_()
    for x in (wide[3:4, 5:134], wide[:, 1:130], wide.t()[:129].t()):
        x = x.detach().requires_grad_()
        assert not x.is_contiguous() or x.shape[0] == 1
        y = linear_8bit(x, w)
        got = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        x2, w2 = x.detach().clone().requires_grad_(), w.detach().contiguous().requires_grad_()
        y2 = linear_8bit(x2, w2)
        want = torch.autograd.grad(y2, (x2, w2), torch.ones_like(y2))
        assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_rms_norm_linear_8bit(gen):
    """The norm and the product in one, against the same of the operators and the gradients' formulas."""
    x, r = (normal(gen, 130, 384).bfloat16().requires_grad_() for _ in range(2))
    nw = (1 + 0.2 * normal(gen, 384)).requires_grad_()
    w = (0.1 * normal(gen, 200, 384)).bfloat16().requires_grad_()
    dy, dt = (0.1 * normal(gen, 130, 200)).bfloat16(), normal(gen, 130, 384).bfloat16()
    y, total = rms_norm_linear_8bit(x, nw, w, r)
    got = torch.autograd.grad((y, total), (x, nw, w, r), (dy, dt))
    with torch.no_grad():
        codes, scales, want_total, rstd = ops.rms_norm_8bit(x, nw, r)
        wc, ws = ops.quantize_8bit(w, BLOCK)
        assert torch.equal(total, want_total) and torch.equal(y, ops.gemm_8bit(codes, scales, wc.t(), ws.t()))
        inner = ops.gemm_8bit(*ops.quantize_8bit(dy), wc, ws)
        dx, dnw = ops.rms_norm_backward(inner, total, nw, rstd, dt)
        normed = ops.rms_norm(total, nw)[0]
        assert torch.equal(got[0], dx) and torch.equal(got[3], dx) and torch.equal(got[1], dnw)
        close(got[2], dy.double().T @ normed.double(), dy.double().abs().T @ normed.double().abs(), 130)
    alone = rms_norm_linear_8bit(x, nw, w)
    alone.sum().backward()
    assert x.grad is not None and r.grad is None
    only = rms_norm_linear_8bit(x, nw, w, r)[1]
    assert torch.autograd.grad(only.sum(), (x, nw, w), allow_unused=True)[1:] == (None, None)


def test_distillation_gradient_against_differences(gen):
    """Central differences along random directions with steps of 2^-6: the third-order term is 2^-12 / 6
    of third derivatives of size one, a loss of size 10 a row errs by 2^-20: both under 1e-3 of the
    sum of magnitudes; the bound is 1e-2 of it."""
    z = normal(gen, 2, 4, 300)
    indices = torch.randint(-1, 300, (2, 4, 12), generator=gen, device=gen.device)
    teacher = normal(gen, 2, 4, 12) * 2
    weight = torch.rand(2, 4, generator=gen, device=gen.device)
    leaf = z.clone().requires_grad_()
    loss = distillation_loss(leaf, indices, teacher, 1.5)
    assert loss.shape == (2, 4) and loss.dtype == torch.float32
    loss.backward(weight)
    for _ in range(4):
        direction, step = normal(gen, *z.shape), 2.0**-6

        def value(sign):
            return (distillation_loss(z + sign * step * direction, indices, teacher, 1.5).double() * weight.double()).sum()

        slope = (value(1) - value(-1)) / (2 * step)
        products = leaf.grad.double() * direction.double()
        assert abs((slope - products.sum()).item()) <= 1e-2 * products.abs().sum().item()


def test_distillation_layer(gen):
    z = normal(gen, 40, 700).bfloat16().requires_grad_()
    indices = torch.randint(-1, 700, (40, 9), generator=gen, device=gen.device)
    teacher = normal(gen, 40, 9).bfloat16()
    distillation_loss(z, indices, teacher).mean().backward()
    even = torch.full((40,), 1 / 40, device=gen.device)
    loss, dlogits = ops.distillation_loss_gradient(even, z.detach(), indices, teacher)
    assert torch.equal(z.grad, dlogits) and torch.equal(loss, distillation_loss(z, indices, teacher))
    none = distillation_loss(z, indices[:, :0], teacher[:, :0])
    assert not none.any() and not torch.autograd.grad(none.sum(), z)[0].any()
    assert distillation_loss(z[:0], indices[:0], teacher[:0]).shape == (0,)


class Together:
    """The output end: norm and product in 8 bits, loss against a teacher's top logits."""

    def __init__(self, gen, rows=150, width=200, vocabulary=1003, top=7):
        self.x, self.stream = (normal(gen, rows, width).bfloat16().requires_grad_() for _ in range(2))
        self.norm = (1 + 0.1 * normal(gen, width)).requires_grad_()
        self.matrix = (0.2 * normal(gen, vocabulary, width)).bfloat16().requires_grad_()
        self.indices = torch.randint(-1, vocabulary, (rows, top), generator=gen, device=gen.device)
        self.indices[::5] = -1
        self.teacher = 2 * normal(gen, rows, top)
        self.leaves = (self.x, self.stream, self.norm, self.matrix)

    def step(self):
        logits, total = rms_norm_linear_8bit(self.x, self.norm, self.matrix, self.stream)
        rows = distillation_loss(logits, self.indices, self.teacher, 2.0)
        return (rows.detach(), *torch.autograd.grad((rows, total), self.leaves, (torch.ones_like(rows), torch.ones_like(total))))

    def renew(self):
        with torch.no_grad():
            self.x.copy_(torch.randn_like(self.x))
            self.matrix.mul_(0.5)
            self.teacher.mul_(-1.0)
            self.indices.copy_(self.indices.flip(0))


def capture(work):
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    return graph, out


def test_run_together(gen):
    """Logits, loss and every gradient of the output end, against the formulas in 64 bits with the codes
    that the operators give. Gradients pass through one 16-bit tensor (the logits', then the norm's):
    each adds half a step of 2^-8 of its own values, which the next product or sum spreads."""
    t = Together(gen)
    rows, dx, dstream, dnorm, dmatrix = t.step()
    with torch.no_grad():
        total = (t.x.float() + t.stream.float()).bfloat16()
        codes, scales, _, rstd = ops.rms_norm_8bit(t.x, t.norm, t.stream)
        spread = scales.double().repeat_interleave(BLOCK, 1)[:, :200]
        w8 = values(t.matrix, BLOCK)
        logits = (codes.double() * spread) @ w8.T
    z = logits.bfloat16().double().requires_grad_()  # as the layer hands them on
    there = t.indices >= 0
    some = there.any(1)
    p = torch.softmax(torch.where(there, t.teacher.double() / 2, -1e300), 1)
    q = torch.log_softmax(z / 2, 1).gather(1, t.indices.clamp_min(0))
    want = 4 * torch.where(there & some[:, None], p * (p.clamp_min(1e-300).log() - q), 0.0).sum(1)
    # Logits may round the other way at a border: half a step of 2^-8 of the largest, in each of the
    # row's logarithms (slope one over T, times T^2).
    slack = 2 * 2.0**-8 * z.detach().abs().amax(1) + 1e-4
    assert ((rows.double() - want.detach()).abs() <= slack).all()
    assert not rows[~some].any()
    (dz,) = torch.autograd.grad(want.sum(), z)
    g8 = values(dz.bfloat16(), 1)
    # Bounds in the 2-norm: each rounding on the way is at most 2^-4 (8 bits) or 2^-8 (16 bits) of the
    # values it meets, and codes differ where a value lies at a border.
    inner = g8 @ w8
    h = total.double() * rstd.double()[:, None]
    a = inner * t.norm.detach().double()
    dtotal = rstd.double()[:, None] * (a - h * (a * h).mean(1, keepdim=True)) + 1
    for got, exact in ((dx, dtotal), (dstream, dtotal), (dnorm, (inner * h).sum(0)),
                       (dmatrix, dz.T @ (h * t.norm.detach().double()))):
        assert ((got.double() - exact).norm() <= 2.0**-5 * exact.norm()).item()


def test_captured_together(gen):
    """Forward and backward in a graph, replayed with other inputs; a second graph of other sizes captured
    and replayed in turn with it; then eager calls again. Each equals the eager step bit for bit."""
    first, second = Together(gen), Together(gen, 40, 136, 70, 3)
    pairs = [(t, *capture(t.step)) for t in (first, second)]
    for t in (first, second):
        t.renew()
    for _ in range(2):
        for _, graph, _ in pairs:
            graph.replay()
    for t, _, captured in pairs:
        for got, want in zip(captured, t.step()):
            assert torch.equal(got, want)


def test_on_other_streams(gen):
    """Two streams at once, each with its own tensors, give what one after the other gives."""
    both = Together(gen), Together(gen, 333, 264, 520, 5)
    want = [t.step() for t in both]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in both]
    got = [None, None]
    for _ in range(3):
        for i, (t, stream) in enumerate(zip(both, streams)):
            with torch.cuda.stream(stream):
                got[i] = t.step()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_types_under_autocast(gen):
    x, w = normal(gen, 4, 64), normal(gen, 64)
    with torch.autocast("cuda", torch.bfloat16):
        assert rms_norm(x, w).dtype == torch.float32
        with pytest.raises(TypeError, match="float16 or bfloat16"):
            linear_8bit(x, x)


def test_muon_steps_the_head(gen):
    """A step of the optimizers on the gradients: Muon's matrix, and the norm's weight with 8-bit moments."""
    t = Together(gen)
    before = t.matrix.detach().clone(), t.norm.detach().clone()
    optimizer = Muon([{"params": [t.matrix]}, {"params": [t.norm], "algorithm": "adamw", "lr": 1e-2, "state_bits": 8}], lr=0.02)
    logits, _ = rms_norm_linear_8bit(t.x, t.norm, t.matrix, t.stream)
    distillation_loss(logits, t.indices, t.teacher).mean().backward()
    optimizer.step()
    for parameter, old in zip((t.matrix, t.norm), before):
        assert torch.isfinite(parameter).all() and not torch.equal(parameter.detach(), old)


def test_example_runs(cuda_device):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    try:
        import distill_head
    finally:
        sys.path.pop(0)
    losses = distill_head.train(steps=4, width=200, vocabulary=1000, tokens=256, top=8)
    assert len(losses) == 4 and all(loss == loss and loss >= 0 for loss in losses)
