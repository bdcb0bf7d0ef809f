"""References for qk_norm_rope and qk_norm_rope_bwd: the RMS norm of every query and key head with the rotation of column
pairs (j, j + half), fp32, and its gradients by autograd of the same expression."""

from __future__ import annotations

import torch


def _angles(cos, sin, positions, batch, seq, sections, interleaved):
    """cos and sin of every token's pairs, [B, S, 1, half]."""
    half = cos.shape[1]
    if positions is None:
        return cos[:seq].expand(batch, seq, half)[:, :, None], sin[:seq].expand(batch, seq, half)[:, :, None]
    rows = positions.long()
    if sections is None:
        return cos[rows][:, :, None], sin[rows][:, :, None]
    axes = len(sections)
    if interleaved:
        axis = [j % axes if j < axes * sections[j % axes] else 0 for j in range(half)]
    else:
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    rows = rows[torch.tensor(axis, device=rows.device)].permute(1, 2, 0)          # [B, S, half]
    pair = torch.arange(half, device=rows.device)
    return cos[rows, pair][:, :, None], sin[rows, pair][:, :, None]


def _forward(x, w, c, s, nope, eps):
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    half = c.shape[-1]
    a, b = n[..., nope:nope + half], n[..., nope + half:nope + 2 * half]
    return torch.cat((n[..., :nope], a * c - b * s, a * s + b * c, n[..., nope + 2 * half:]), -1)


def qk_norm_rope_ref(q, k, q_weight, k_weight, cos, sin, positions=None, eps: float = 1e-6, nope_dim=None, sections=None,
                     interleaved: bool = False):
    nope = q.shape[3] - 2 * cos.shape[1] if nope_dim is None else nope_dim
    c, s = _angles(cos, sin, positions, q.shape[0], q.shape[1], sections, interleaved)
    return [_forward(x.float(), w.float(), c, s, nope, eps).to(x.dtype) for x, w in ((q, q_weight), (k, k_weight))]


def qk_norm_rope_bwd_ref(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, positions=None, eps: float = 1e-6, nope_dim=None,
                         sections=None, interleaved: bool = False):
    nope = q.shape[3] - 2 * cos.shape[1] if nope_dim is None else nope_dim
    c, s = _angles(cos, sin, positions, q.shape[0], q.shape[1], sections, interleaved)
    grads, weights = [], []
    for dy, x, w in ((dq_out, q, q_weight), (dk_out, k, k_weight)):
        xf, wf = x.float().requires_grad_(), w.float().requires_grad_()
        with torch.enable_grad():
            gx, gw = torch.autograd.grad(_forward(xf, wf, c, s, nope, eps), (xf, wf), dy.float())
        grads.append(gx.to(x.dtype))
        weights.append(gw.to(w.dtype))
    return grads + weights
