"""Checker of add_rms_norm_quant: the residual sum rounded to the inputs' type, its RMS norm with the weight
in fp32, and e4m3 values with one scale per group of columns (the group's largest magnitude is held as 448)."""

from __future__ import annotations

import torch

E4M3_MAX = 448.0
TINY = 2.0 ** -100


def add_rms_norm_quant_ref(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6,
                           group: int | None = 128):
    n = x.shape[-1]
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hf = h.float().view(-1, n)
    inv_rms = 1 / (hf.square().mean(-1, keepdim=True) + eps).sqrt()
    u = (hf * weight.float()).view(hf.shape[0], -1, group or n)
    a = u.abs().amax(-1).clamp_min(TINY)
    qmax = torch.full_like(a, E4M3_MAX)  # tensor / tensor: torch divides a tensor by a number through its reciprocal
    y = (u * (qmax / a)[..., None]).to(torch.float8_e4m3fn)
    scale = a * inv_rms / qmax
    return y.view(x.shape), scale.t().contiguous() if group else scale.view(-1), h
