"""Differentiable layers on the B200 kernels: a layer norm and a linear layer of experts.

``layer_norm`` and ``grouped_linear`` run forward and backward in the kernels behind
``ops.layer_norm`` and ``ops.grouped_gemm`` and work with torch's autograd. An expert
layer's weights [experts, out, in] are a batch of matrices as the orthogonaliser takes it,
so ``Muon`` steps them in one call; the norms, routers and embeddings beside them go to
an ``adamw`` group, whose moments may be held in 8 bits (``"state_bits": 8``). The
reference has no layers; these are what its optimizers are used next to.

They run eagerly and in captured CUDA graphs. ``torch.compile`` breaks its graph at each of
them (``fullgraph=True`` refuses), there is no forward mode and no ``vmap``, and they do not
cast under autocast: ``grouped_linear`` refuses fp32 inputs there as elsewhere.
"""

from __future__ import annotations

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
