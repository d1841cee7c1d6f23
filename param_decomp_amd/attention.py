"""Causal attention over packed sequences with grouped heads, on the GPU.

The attention between a language-model target's decomposed projections
(`param_decomp/param_decomp/attention.py:26-130`), for a token axis that holds several
sequences: `q`, `k` and `v` are what `site_forward` gives for q_proj, k_proj and v_proj
(after any rotary rotation), the result is what o_proj reads. The stack step `lm_step` has
its own form for equal-length batches inside.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from param_decomp_amd import ops


def _dense(t: torch.Tensor) -> torch.Tensor:
    """The tensor, or a dense copy where its rows or heads are not 16-byte aligned or its
    rows are more than 8 MiB apart."""
    per = 16 // t.element_size()
    if t.dim() == 3 and t.numel() and (t.stride(2) != 1 or t.stride(0) % per or t.stride(1) % per or
                                       t.data_ptr() % 16 or t.stride(0) * t.element_size() > 1 << 23):
        return t.clone(memory_format=torch.contiguous_format)
    return t


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, scale):
        out, (stats, rest) = ops.packed_attention_fwd(q, k, v, offsets, scale=scale, want_saved=True)
        ctx.save_for_backward(q, k, v, offsets, out, stats, rest)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, offsets, out, stats, rest = ctx.saved_tensors
        dq, dk, dv = ops.packed_attention_bwd(q, k, v, offsets, out, (stats, rest), _dense(g.contiguous()),
                                              scale=ctx.scale)
        return dq, dk, dv, None, None


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, *,
                     scale: float | None = None) -> torch.Tensor:
    """Row i of sequence [offsets[s], offsets[s + 1]) attends to the sequence's rows up to
    itself: q [rows, H, head_dim], k and v [rows, KV, head_dim], bf16 or fp32 (views of one
    projection's output are read as they are), H a multiple of KV, head_dim up to 128;
    offsets int32 [sequences + 1] on the same GPU. Returns [rows, H, head_dim], zeros in
    rows of no sequence; differentiable in q, k and v (not in forward mode, and once). Scores
    and sums are fp32; bf16 operands meet weights rounded to bf16. `scale`: head_dim^-0.5 by
    default."""
    D = q.shape[-1] if q.dim() else 0
    pad = (-D) % 8
    if pad and D <= 128:  # zero columns add nothing to the scores and are cut off the result
        if scale is None:
            scale = D**-0.5
        q, k, v = (torch.nn.functional.pad(t, (0, pad)) for t in (q, k, v))
        return packed_attention(q, k, v, offsets, scale=scale)[..., :D]
    q, k, v = _dense(q), _dense(k), _dense(v)
    if ops.differentiated(q, k, v):
        return _PackedAttention.apply(q, k, v, offsets, scale)
    return ops.packed_attention_fwd(q, k, v, offsets, scale=scale)[0]
