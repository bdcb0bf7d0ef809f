"""qk_norm_rope_bwd plugin module: the gradients of ``qk_norm_rope``, with the module contract of the reference's
plugins (``kernels/__init__.py:3-8``).  The reference has no backward pass.

    kernel_fn(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, positions=None, *, eps=1e-6, nope_dim=None,
              sections=None, interleaved=False) -> (dq, dk, dq_weight, dk_weight)

dq_out, dk_out are the gradients of the forward's outputs, shaped and typed like q and k; everything else as the forward
took it (nothing needs to be kept from it).  With r = 1 / sqrt(mean(x^2) + eps) and g the gradient turned back by the
position's angles:

    dweight = sum over rows of g x r,    dx = r (g weight - x r^2 mean(g weight x))

fp32 arithmetic.  dq, dk are contiguous in the type of q; the weights' gradients are summed over all tokens and heads in fp32 in
an order that the sizes and the GPU's number of SMs decide (the same bits every time) and rounded to the weights' type.

``kernel_fn`` runs ``tokmix_qk_norm_rope_bwd`` (``csrc/qk_norm_rope.cu``), no fallback."""

from __future__ import annotations

import functools

import torch

from . import _lib
from . import qk_norm_rope as _forward
from .qk_norm_rope import check_device_status  # noqa: F401

KERNEL_TYPE = "qk_norm_rope_bwd"


@functools.lru_cache(maxsize=256)
def _workspace_bytes(tokens: int, heads_q: int, heads_k: int, head_dim: int, device: torch.device) -> int:
    return _lib.call_on(device, _lib.load().tokmix_qk_norm_rope_bwd_workspace_bytes, tokens, heads_q, heads_k, head_dim)


def kernel_fn(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,
              k_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None = None, *,
              eps: float = 1e-6, nope_dim: int | None = None, sections: tuple | None = None, interleaved: bool = False):
    args, dq, dk, keep = _forward.describe(q, k, q_weight, k_weight, cos, sin, positions, eps, nope_dim, sections, interleaved,
                                           (dq_out, dk_out))
    dev = q.device
    dqw, dkw = torch.empty_like(keep[2]), torch.empty_like(keep[3])
    batch, seq, hq, d = q.shape
    need = _workspace_bytes(batch * seq, hq, k.shape[2], d, dev)
    ws = _lib.empty((need or 1,), torch.uint8, dev)  # per call: calls may overlap on other streams
    status = _lib.host_status_ptr(dev, "qk_norm_rope")
    rc = _lib.call_on(dev, _lib.load().tokmix_qk_norm_rope_bwd, args, dqw.data_ptr(), dkw.data_ptr(), ws.data_ptr(),
                      need, status, _lib.stream_ptr(dev))
    del keep
    if rc:
        _lib.check(rc, "qk_norm_rope_bwd")
    _lib.after_host_status_launch(dev, "qk_norm_rope")
    return dq, dk, dqw, dkw


def get_inputs(batch: int = 4, seq_len: int = 2048, q_heads: int = 16, kv_heads: int = 2, head_dim: int = 256,
               pairs: int = 32, dtype: torch.dtype = torch.bfloat16, seed: int = 42, device: str = "cuda") -> dict:
    inp = _forward.get_inputs(batch, seq_len, q_heads, kv_heads, head_dim, pairs, dtype, seed, device)
    gen = torch.Generator().manual_seed(seed + 1)
    return {"dq_out": torch.randn(inp["q"].shape, generator=gen).to(dtype).to(device),
            "dk_out": torch.randn(inp["k"].shape, generator=gen).to(dtype).to(device), **inp}


def get_flops(batch: int = 4, seq_len: int = 2048, q_heads: int = 16, kv_heads: int = 2, head_dim: int = 256) -> int:
    return 16 * batch * seq_len * (q_heads + kv_heads) * head_dim


def get_bytes(batch: int = 4, seq_len: int = 2048, q_heads: int = 16, kv_heads: int = 2, head_dim: int = 256,
              pairs: int = 32, element_size: int = 2) -> int:
    """q, k and the outputs' gradients read, dq and dk written once; tables, weights and their gradients once."""
    return (batch * seq_len * (q_heads + kv_heads) * head_dim * element_size * 3 + seq_len * pairs * 8
            + 4 * head_dim * element_size)
