"""Layer norm on the GPU, forward and backward (fp32 statistics and parameter gradients)."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from param_decomp_amd import ops


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = ops.layer_norm_fwd(x, weight, bias, eps=eps, want_stats=True)
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, stats = ctx.saved_tensors
        want = ctx.needs_input_grad
        return (*ops.layer_norm_bwd(x, g.contiguous(), weight, stats, want_dx=want[0], want_dweight=want[1],
                                    want_dbias=want[2]), None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """`(x - mean) / sqrt(var + eps) * weight + bias` over the last axis: x bf16 or fp32
    [..., d], weight and bias fp32 [d] (None: 1 and 0), as the stack steps keep norm weights.
    Differentiable in all three."""
    x = x.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if ops.differentiated(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return ops.layer_norm_fwd(x, weight, bias, eps=eps)[0]
