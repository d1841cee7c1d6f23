"""Norms on the GPU, forward and backward (fp32 statistics and parameter gradients): layer norm, and
the RMS norms before and after a residual branch with its gate and scale."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from param_decomp_amd import _lib as L
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


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, post_weight, gate, pre_weight, opts, eps):
        ctx.set_materialize_grads(False)
        h, y, stats = ops.residual_norm_fwd(x, branch, post_weight=post_weight, gate=gate, pre_weight=pre_weight, eps=eps,
                                            want_stats=True, **opts)
        ctx.save_for_backward(h, branch, post_weight, gate, pre_weight, stats)
        ctx.opts = opts
        return y if branch is None else (h, y)

    @staticmethod
    @once_differentiable
    def backward(ctx, *g):
        h, branch, post_weight, gate, pre_weight, stats = ctx.saved_tensors
        gh, gy = g if branch is not None else (None, g[0])
        want = ctx.needs_input_grad
        if gh is None and gy is None:
            return (None,) * 7
        dx, db, dpost, dg, dpre = ops.residual_norm_bwd(
            h, branch, stats, None if gh is None else gh.contiguous(), None if gy is None else gy.contiguous(),
            post_weight=post_weight, gate=gate, pre_weight=pre_weight, want_dx=want[0], want_dbranch=want[1],
            want_dpost=want[2], want_dgate=want[3], want_dpre=want[4], **ctx.opts)
        return dx, db, dpost, dg, dpre, None, None


def _dense(t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else t.contiguous()


def _gate_rows(x: torch.Tensor, gate: torch.Tensor) -> None:
    """Refuses a gate whose rows are not those of leading axes of x (or of runs of a flat x's rows)."""
    lead = gate.shape[:-1]
    while lead and lead[-1] == 1:
        lead = lead[:-1]
    if lead != x.shape[:len(lead)] and not (x.dim() == 2 and len(lead) == 1 and lead[0] and x.shape[0] % lead[0] == 0) or \
            gate.dim() > x.dim():
        raise L.PDError(f"residual_norm: a gate {tuple(gate.shape)} does not go by the leading axes of {tuple(x.shape)}")


def residual_norm(x: torch.Tensor, branch: torch.Tensor, *, post_norm: bool = True,
                  post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  pre_weight: torch.Tensor | None = None, scale: float = 1.0, zero_centered: bool = False,
                  eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """What lies between two branches of a residual stream, in one pass: `stream = x + scale * gate *
    rms_norm(branch, post_weight)` and `y = rms_norm(stream, pre_weight)`, the next branch's input.
    Returns (stream, y).

    x [..., d] bf16 or fp32, branch of its shape (bf16 with an fp32 stream too), y in the branch's
    dtype; weights fp32 [d] (None: 1; `zero_centered`: 1 + weight, as
    `param_decomp/param_decomp/targets/qwen36_moe.py` keeps them). `post_norm` False leaves the branch
    as it is. gate [d] (channels), or fp32 or bf16 [..., d] over leading axes of x: [batch, d] or
    [batch, 1, d] for x [batch, T, d], or x's own shape; for x [rows, d] any [n, d] whose n divides
    the rows, each for rows / n rows in turn. y norms the stream as stored, in x's
    dtype. d up to 16384. Differentiable in the five tensors, once."""
    if gate is not None:
        _gate_rows(x, gate)
    opts = dict(post_norm=bool(post_norm), scale=float(scale), weight_offset=1.0 if zero_centered else 0.0)
    args = [_dense(t) for t in (x, branch, post_weight, gate, pre_weight)]
    if ops.differentiated(*args):
        return _ResidualNorm.apply(*args, opts, eps)
    x, branch, post_weight, gate, pre_weight = args
    return ops.residual_norm_fwd(x, branch, post_weight=post_weight, gate=gate, pre_weight=pre_weight, eps=eps, **opts)[:2]


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, *, zero_centered: bool = False, eps: float = 1e-6,
             dtype: torch.dtype | None = None) -> torch.Tensor:
    """`x / sqrt(mean(x^2) + eps) * weight` over the last axis, the norm in front of the first
    branch: x bf16 or fp32 [..., d], d up to 16384, the result in `dtype` (x's by default, bf16 of an
    fp32 x). Differentiable in both, once."""
    opts = dict(post_norm=False, weight_offset=1.0 if zero_centered else 0.0, y_dtype=dtype or x.dtype)
    x, weight = _dense(x), _dense(weight)
    if ops.differentiated(x, weight):
        return _ResidualNorm.apply(x, None, None, None, weight, opts, eps)
    return ops.residual_norm_fwd(x, None, pre_weight=weight, eps=eps, **opts)[1]
