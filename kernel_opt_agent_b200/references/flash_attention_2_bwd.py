"""Reference for flash_attention_2_bwd: the gradients in fp32 from the inputs, the output and the log-sum-exp, one
key/value head at a time."""

from __future__ import annotations

import math

import torch


def flash_attention_2_bwd_ref(do, q, k, v, o, lse, causal: bool = True, sm_scale: float | None = None, layout: str = "bhsd"):
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(q.shape[-1])
    grads = [torch.empty_like(t) for t in (q, k, v)]
    first = (lambda t: t) if layout == "bhsd" else (lambda t: t.transpose(1, 2))
    do, q, k, v, o = (first(t) for t in (do, q, k, v, o))
    dq, dk, dv = (first(t) for t in grads)
    group = q.shape[1] // k.shape[1]
    for b in range(q.shape[0]):
        for h in range(k.shape[1]):
            heads = slice(h * group, (h + 1) * group)
            qf, dof, kf, vf = q[b, heads].float(), do[b, heads].float(), k[b, h].float(), v[b, h].float()
            p = torch.exp(qf @ kf.T * sm_scale - lse[b, heads, :, None])
            if causal:
                p = p.masked_fill(torch.ones(p.shape[1:], dtype=torch.bool, device=p.device).triu(1), 0.0)
            dv[b, h] = (p.flatten(0, 1).T @ dof.flatten(0, 1)).to(dv.dtype)
            ds = p * (dof @ vf.T - (dof * o[b, heads].float()).sum(-1, keepdim=True)) * sm_scale
            dq[b, heads] = (ds @ kf).to(dq.dtype)
            dk[b, h] = (ds.flatten(0, 1).T @ qf.flatten(0, 1)).to(dk.dtype)
    return grads
