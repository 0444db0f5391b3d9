"""Differentiable layers on the B200 kernels: norms, linear layers and a loss.

``layer_norm`` and ``grouped_linear`` run forward and backward in the kernels behind
``ops.layer_norm`` and ``ops.grouped_gemm`` and work with torch's autograd; so do
``rms_norm``, ``linear_8bit`` (products in 8 bits with scales for blocks of 128),
``rms_norm_linear_8bit`` (the two of them, with the norm written in 8 bits) and
``distillation_loss``. An expert layer's weights [experts, out, in] are a batch of matrices as
the orthogonaliser takes it, so ``Muon`` steps them in one call; the norms, routers and
embeddings beside them go to an ``adamw`` group, whose moments may be held in 8 bits
(``"state_bits": 8``). The reference has no layers; these are what its optimizers are used
next to.

They run eagerly and in captured CUDA graphs. ``torch.compile`` breaks its graph at each of
them (``fullgraph=True`` refuses), there is no forward mode and no ``vmap``, and they do not
cast under autocast: ``grouped_linear`` and the 8-bit layers refuse fp32 inputs there as
elsewhere.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from gram_newton_schulz_ampere_b200 import ops


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, bias: Tensor | None, epsilon: float) -> Tensor:  # type: ignore[no-untyped-def]
        y, mean, rstd = ops.layer_norm(x, weight, bias, epsilon)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):  # type: ignore[no-untyped-def]
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dweight, dbias = ops.layer_norm_backward(grad, x, weight, mean, rstd)
        needs = ctx.needs_input_grad
        return dx if needs[0] else None, dweight if needs[1] else None, dbias if needs[2] else None, None


def layer_norm(x: Tensor, weight: Tensor, bias: Tensor | None = None, epsilon: float = 1e-5) -> Tensor:
    """Layer norm over the last dimension of x, differentiable in x, weight and bias.

    x is float16, bfloat16 or float32 of any shape and strides; weight and bias (which may be
    None) share a type of their own. Statistics and sums are fp32. The backward pass reads x
    and the gradient once and sums the weight's gradient in a fixed order."""
    return _LayerNorm.apply(x, weight, bias, epsilon)


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, ends: Tensor) -> Tensor:  # type: ignore[no-untyped-def]
        ctx.save_for_backward(x, weight, ends)
        return ops.grouped_gemm(x, weight.transpose(1, 2), ends)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):  # type: ignore[no-untyped-def]
        x, weight, ends = ctx.saved_tensors
        grad = ops.row_operand(grad)  # a copy for TMA, if one is needed, is made once
        dx = ops.grouped_gemm(grad, weight, ends) if ctx.needs_input_grad[0] else None
        dweight = ops.grouped_gemm_reduce(grad, x, ends) if ctx.needs_input_grad[1] else None
        return dx, dweight, None


def grouped_linear(x: Tensor, weight: Tensor, ends: Tensor) -> Tensor:
    """``y[r] = x[r] @ weight[e].T`` for the rows r of each expert e, differentiable in x and weight.

    x [rows, in] holds the rows sorted by expert, weight [experts, out, in] one matrix for each
    (float16 or bfloat16, as x); ``ends`` [experts] are the row numbers where the experts' rows
    end (int32 or int64, on the device; see ``ops.grouped_gemm``). Rows past the last end give
    zeros and get zero gradients; an expert without rows gets a zero gradient. Nothing is read
    back to the host."""
    if weight.ndim != 3:
        raise ValueError("expected weight [experts, out, in]")
    return _GroupedLinear.apply(x, weight, ends)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, residual: Tensor | None, epsilon: float):  # type: ignore[no-untyped-def]
        y, total, rstd = ops.rms_norm(x, weight, residual, epsilon)
        ctx.save_for_backward(total, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor | None, grad_total: Tensor | None = None):  # type: ignore[no-untyped-def]
        total, weight, rstd = ctx.saved_tensors
        needs = ctx.needs_input_grad
        dx, dweight = grad_total, None
        if grad is not None:
            dx, dweight = ops.rms_norm_backward(grad, total, weight, rstd, grad_total)
        return dx if needs[0] else None, dweight if needs[1] else None, dx if needs[2] else None, None


def rms_norm(
    x: Tensor, weight: Tensor, residual: Tensor | None = None, epsilon: float = 1e-5
) -> Tensor | tuple[Tensor, Tensor]:
    """Root-mean-square norm over the last dimension, differentiable in x, weight and residual.

    Without a residual, the norm of x. With one (the residual stream that x, a layer's output,
    is added to), the norm of ``x + residual`` and that sum, the stream as the next layer takes
    it. Types as for ``ops.rms_norm``."""
    return _RmsNorm.apply(x, weight, residual, epsilon)


def _check_16_bits(x: Tensor, weight: Tensor) -> None:
    if weight.ndim != 2 or weight.numel() == 0 or x.ndim < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError("expected x [..., in] and weight [out, in], neither size zero")
    if x.dtype != weight.dtype or x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("x and weight must share dtype float16 or bfloat16")


def _weight_gradient(grad: Tensor, x: Tensor) -> Tensor:
    """``grad.T @ x`` of 16-bit matrices [rows, out] and [rows, in]."""
    if grad.shape[0] == 0:
        return grad.new_zeros((grad.shape[1], x.shape[1]))
    return ops._rows_product(grad, x)


class _Linear8bit(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor) -> Tensor:  # type: ignore[no-untyped-def]
        y, kept = ops._linear_8bit(x, weight)
        # x serves the weight's gradient, the weight's codes that of x.
        needs_x, needs_weight = ctx.needs_input_grad
        ctx.save_for_backward(x if needs_weight else None, kept if needs_x else None)
        ctx.x_shape = x.shape
        ctx.shape = n, _ = weight.shape
        return y if x.ndim == 2 else y.view(*x.shape[:-1], n)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):  # type: ignore[no-untyped-def]
        x, kept = ctx.saved_tensors
        n, k = ctx.shape
        grad = grad.reshape(-1, n)
        dx = dweight = None
        if ctx.needs_input_grad[0]:
            dx = ops._linear_8bit_gradient(grad, kept, n, k).view(ctx.x_shape)
        if ctx.needs_input_grad[1]:
            dweight = _weight_gradient(grad, x.reshape(-1, k))
        return dx, dweight


def linear_8bit(x: Tensor, weight: Tensor) -> Tensor:
    """``x @ weight.T`` with both factors in 8 bits, differentiable in x and weight.

    x [..., in] and weight [out, in] share float16 or bfloat16, and so do the result and the
    gradients. Each call brings x (a scale for each 128 of a row) and the weight (a scale for each
    128 x 128 block) into e4m3; the backward pass does so with the output's gradient for the
    gradient of x, against the codes of the forward pass. The weight's gradient is the product
    of the 16-bit gradient and x: what is rounded to 8 bits on the way to it is nothing."""
    _check_16_bits(x, weight)
    return _Linear8bit.apply(x, weight)


class _RmsNormLinear8bit(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, norm_weight, weight, residual, epsilon):  # type: ignore[no-untyped-def]
        normed, scale, total, rstd = ops.rms_norm_8bit(x, norm_weight, residual, epsilon)
        codes, scales = ops.quantize_8bit(weight, 128)
        y = ops.gemm_8bit(normed, scale, codes.t(), scales.t(), out_dtype=x.dtype)
        # The weight's gradient takes the stream and the norm's weight; all others pass through the product.
        needs = ctx.needs_input_grad
        through = (rstd, codes, scales) if needs[0] or needs[1] or needs[3] else (None, None, None)
        ctx.save_for_backward(total, norm_weight, *through)
        ctx.set_materialize_grads(False)
        ctx.epsilon = epsilon
        ctx.shape = weight.shape
        y = y.view(*x.shape[:-1], weight.shape[0])
        return y if residual is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, grad_total=None):  # type: ignore[no-untyped-def]
        total, norm_weight, rstd, codes, scales = ctx.saved_tensors
        needs = ctx.needs_input_grad
        n, k = ctx.shape
        dx, dnorm, dweight = grad_total, None, None
        if grad is not None:
            grad = grad.reshape(-1, n)
            if needs[0] or needs[1] or needs[3]:
                inner = ops.gemm_8bit(*ops.quantize_8bit(grad), codes, scales, out_dtype=total.dtype)
                dx, dnorm = ops.rms_norm_backward(inner.view(total.shape), total, norm_weight, rstd, grad_total)
            if needs[2]:
                # The norm is made again in 16 bits: cheaper than keeping it.
                normed = ops.rms_norm(total, norm_weight, None, ctx.epsilon)[0]
                dweight = _weight_gradient(grad, normed.view(-1, k))
        return dx if needs[0] else None, dnorm if needs[1] else None, dweight, dx if needs[3] else None, None


def rms_norm_linear_8bit(
    x: Tensor, norm_weight: Tensor, weight: Tensor, residual: Tensor | None = None, epsilon: float = 1e-5
) -> Tensor | tuple[Tensor, Tensor]:
    """``linear_8bit(rms_norm(x, norm_weight, residual), weight)`` with the norm written in 8 bits
    only, differentiable in all four. Returns what ``rms_norm`` does, the layer's output in the
    norm's place. The weight's gradient takes the norm in 16 bits, made again from the stream."""
    _check_16_bits(x, weight)
    return _RmsNormLinear8bit.apply(x, norm_weight, weight, residual, epsilon)


class _DistillationLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, indices: Tensor, teacher: Tensor, temperature: float) -> Tensor:  # type: ignore[no-untyped-def]
        loss, statistics = ops.distillation_loss(logits, indices, teacher, temperature)
        ctx.save_for_backward(logits, indices, teacher, statistics)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):  # type: ignore[no-untyped-def]
        logits, indices, teacher, statistics = ctx.saved_tensors
        dlogits = ops.distillation_loss_backward(grad, logits, indices, teacher, statistics, ctx.temperature)
        return dlogits, None, None, None


def distillation_loss(logits: Tensor, indices: Tensor, teacher: Tensor, temperature: float = 1.0) -> Tensor:
    """The fp32 loss of each row against a teacher's top logits, differentiable in the logits.

    logits [..., vocabulary], indices and teacher [..., top]: which logits the teacher gives and
    what they are (``ops.distillation_loss`` has the formula and what is left out; -1 marks an
    entry, and a row of -1 a token, that has no part). The backward pass reads the logits again
    and writes their gradient; a loop that knows each row's weight beforehand saves a reading
    with ``ops.distillation_loss_gradient``."""
    if teacher.requires_grad:
        raise ValueError("the teacher's logits get no gradient: pass them detached")
    if logits.shape[:-1] != indices.shape[:-1] or indices.shape != teacher.shape or logits.ndim < 1:
        raise ValueError("expected logits [..., vocabulary] and indices and teacher [..., top]")
    rows, top = math.prod(logits.shape[:-1]), indices.shape[-1]
    loss = _DistillationLoss.apply(logits.reshape(rows, logits.shape[-1]), indices.reshape(rows, top),
                                   teacher.reshape(rows, top), temperature)
    return loss.view(logits.shape[:-1])
