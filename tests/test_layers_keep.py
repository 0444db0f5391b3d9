"""What the differentiable 8-bit layers keep for their backward pass, and that it is what the pass
reads: on the CPU with the kernels' calls replaced by plain ones of the same results' shapes, and on
the kernels."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops, training

ROWS, K, N = 6, 10, 7


def norm(x, weight, residual, epsilon):
    total = x if residual is None else x + residual
    rstd = (total.float().square().mean(-1) + epsilon).rsqrt()
    return (total * rstd[..., None].to(x.dtype) * weight.to(x.dtype)), total, rstd


@pytest.fixture
def plain(monkeypatch):
    def norm_8bit(x, weight, residual, epsilon):
        y, total, rstd = norm(x, weight, residual, epsilon)
        return y.reshape(-1, K), torch.ones(1, 1), total, rstd

    def norm_backward(grad, total, weight, rstd, grad_total=None):
        return grad.clone() if grad_total is None else grad + grad_total, torch.ones_like(weight)

    def quantize(x, block_rows=1):
        return x, torch.ones(1, 1)

    def gemm(left, left_scales, right, right_scales, out_dtype=torch.bfloat16):
        return (left.float() @ right.float()).to(out_dtype)

    def linear(x, weight):
        return (x.reshape(-1, K).float() @ weight.float().t()).to(x.dtype), weight.detach().clone()

    def linear_gradient(grad, kept, n, k):
        return (grad.float() @ kept.float()).to(grad.dtype)

    def rows_product(left, right):
        return (left.float().t() @ right.float()).to(left.dtype)

    for name, call in (("rms_norm", norm), ("rms_norm_8bit", norm_8bit), ("rms_norm_backward", norm_backward),
                       ("quantize_8bit", quantize), ("gemm_8bit", gemm), ("_linear_8bit", linear),
                       ("_linear_8bit_gradient", linear_gradient), ("_rows_product", rows_product)):
        monkeypatch.setattr(ops, name, call)


def kept(call):
    """The elements that `call` keeps, and its result."""
    sizes = []

    def pack(t):
        sizes.append(t.numel())
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        out = call()
    return sum(sizes), out


def leaf(needs, *shape):
    return torch.randn(shape).bfloat16().requires_grad_(needs)


@pytest.mark.parametrize("x_needs,w_needs", [(True, True), (True, False), (False, True)])
def test_linear(plain, x_needs, w_needs):
    x, w = leaf(x_needs, 2, ROWS, K), leaf(w_needs, N, K)
    elements, y = kept(lambda: training.linear_8bit(x, w))
    assert elements == (N * K if x_needs else 0) + (2 * ROWS * K if w_needs else 0)
    y.sum().backward()
    for t, needs in ((x, x_needs), (w, w_needs)):
        assert (t.grad is not None) == needs and (not needs or t.grad.shape == t.shape)


@pytest.mark.parametrize("x_needs,norm_needs,w_needs,r_needs", [
    (True, True, True, True), (True, False, False, False), (False, True, False, False), (False, False, True, False),
    (False, False, False, True), (False, True, True, False), (True, True, False, None), (False, False, True, None),
])
def test_norm_and_linear(plain, x_needs, norm_needs, w_needs, r_needs):
    x, nw, w = leaf(x_needs, 2, ROWS, K), leaf(norm_needs, K), leaf(w_needs, N, K)
    r = None if r_needs is None else leaf(r_needs, 2, ROWS, K)
    elements, out = kept(lambda: training.rms_norm_linear_8bit(x, nw, w, r))
    through = x_needs or norm_needs or bool(r_needs)
    # The stream and the norm's weight serve both; codes, their scale and rstd the norm's gradient alone.
    assert elements == 2 * ROWS * K + K + (N * K + 1 + 2 * ROWS if through else 0)
    y = out if r is None else out[0]
    assert y.shape == (2, ROWS, N)
    y.sum().backward()
    for t, needs in ((x, x_needs), (nw, norm_needs), (w, w_needs), (r, bool(r_needs))):
        if t is not None:
            assert (t.grad is not None) == needs and (not needs or t.grad.shape == t.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("residual", [False, True])
def test_gradients_of_any_subset_are_those_of_all(cuda_device, residual):
    """The kernels' layers with every choice of frozen inputs: the same bits as with none frozen."""
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    shapes = [(3, 50, 136), (136,), (200, 136)] + ([(3, 50, 136)] if residual else [])
    values = [torch.randn(shape, generator=gen, device=cuda_device).bfloat16() for shape in shapes]
    dy = torch.randn(3, 50, 200, generator=gen, device=cuda_device).bfloat16()

    def gradients(call, needs):
        leaves = [v.clone().requires_grad_(n) for v, n in zip(values, needs)]
        out = call(leaves)
        (out[0] if isinstance(out, tuple) else out).backward(dy)
        return [t.grad for t in leaves]

    places = range(len(shapes))
    for call, inputs in ((lambda t: training.rms_norm_linear_8bit(*t), set(places)),
                         (lambda t: training.linear_8bit(t[0], t[2]), {0, 2})):
        whole = gradients(call, [True for _ in places])
        for bits in range(1, 2 ** len(shapes)):
            needs = [bool(bits >> i & 1) for i in places]
            if not any(needs[i] for i in inputs):
                continue
            for i, (got, want) in enumerate(zip(gradients(call, needs), whole)):
                assert (got is not None) == (needs[i] and i in inputs)
                assert got is None or torch.equal(got, want)
