"""The attention layer's kernels behind autograd: calls that a training step differentiates through.

    q, k = training.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, ...)
    o = training.attention(q, k, v, causal=True, layout="bshd")
    loss(o).backward()

Each is its plugin modules' ``kernel_fn`` (``qk_norm_rope`` and ``qk_norm_rope_bwd``, ``flash_attention_2`` and
``flash_attention_2_bwd``), with their arguments, checks and errors; cos, sin and positions get no gradient.  The gradients
are those of the first order only, in contiguous tensors.  Between the passes attention keeps q, k, v (copies of those that are not
contiguous), its output and one fp32 number per row, qk_norm_rope its inputs.

A step that is to be captured into a CUDA graph makes its first calls before the capture (as every module here), and its
autograd graph inside it; a graph of the same leaves that was built outside should be gone by then (autograd accumulates on
the stream on which a leaf's graph was first built, which a capture cannot join).  ``kernel_fn`` of the four modules has no
such condition."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import flash_attention_2, flash_attention_2_bwd, qk_norm_rope_bwd
from . import qk_norm_rope as _norm


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, sm_scale, layout):
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()  # as the kernels read them, in both passes
        o, lse = flash_attention_2.kernel_fn(q, k, v, causal, sm_scale, layout=layout, return_lse=True)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.options = (causal, sm_scale)
        ctx.layout = layout
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse = ctx.saved_tensors
        grads = flash_attention_2_bwd.kernel_fn(do, q, k, v, o, lse, *ctx.options, layout=ctx.layout)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True, sm_scale: float | None = None, *,
              layout: str = "bhsd") -> torch.Tensor:
    """``flash_attention_2.kernel_fn`` with gradients for q, k and v."""
    return _Attention.apply(q, k, v, causal, sm_scale, layout)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, options):
        out = _norm.kernel_fn(q, k, q_weight, k_weight, cos, sin, positions, **options)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.options = options
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        grads = qk_norm_rope_bwd.kernel_fn(dq_out, dk_out, *ctx.saved_tensors, **ctx.options)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None, None)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, positions: torch.Tensor | None = None, *, eps: float = 1e-6,
                 nope_dim: int | None = None, sections: tuple | None = None, interleaved: bool = False):
    """``qk_norm_rope.kernel_fn`` with gradients for q, k and both weights."""
    return _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions,
                             dict(eps=eps, nope_dim=nope_dim, sections=sections, interleaved=interleaved))
