"""flash_attention_2_bwd plugin module: the gradients of ``flash_attention_2``, with the module contract
of the reference's plugins (``kernels/__init__.py:3-8``).  The reference has no backward pass.

    kernel_fn(do, q, k, v, o, lse, causal=True, sm_scale=None, *, layout="bhsd") -> (dq, dk, dv)

q, k, v, causal, sm_scale and layout as the forward took them; o and lse what it returned with
``return_lse=True``; do the gradient of o, shaped like it.  All bf16, lse fp32 [batch, heads, seq] (in
both layouts).  With P = exp(sm_scale q k^T - lse) under the mask and delta = sum(do * o) per row:

    dv = P^T do,   dS = P * (do v^T - delta),   dq = sm_scale dS k,   dk = sm_scale dS^T q

dk and dv are summed over the query heads that share a key/value head.  P and dS enter their products in
bf16, sums are fp32, and every sum has an order that the sizes and the GPU's number of SMs decide: the same bits every time.
A key or value that no query sees gets zeros.  What is masked is replaced in P and dS, whose products are then taken whole: a value
of v that is not finite stays out of the rows that do not see it, one of q, k or do can reach other rows of its tile.
Tensors that are not contiguous (a gradient that autograd expanded, say) are copied first.

``kernel_fn`` runs ``tokmix_fa2_bwd`` (``csrc/fa2_bwd.cu``), no fallback.  ``training.attention`` is the forward
and this in one differentiable call."""

from __future__ import annotations

import functools
import math

import torch

from . import _lib
from . import flash_attention_2 as _forward

KERNEL_TYPE = "flash_attention_2_bwd"


@functools.lru_cache(maxsize=256)
def _workspace_bytes(batch: int, heads: int, heads_kv: int, sq: int, skv: int, d: int, causal: int, device: torch.device) -> int:
    need = _lib.call_on(device, _lib.load().tokmix_fa2_bwd_workspace_bytes, batch, heads, heads_kv, sq, skv, d, causal)
    return max(need, 0)  # bad sizes: the call itself says which


def kernel_fn(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
              causal: bool = True, sm_scale: float | None = None, *, layout: str = "bhsd"):
    q, k, v, hd, sd = _forward._validate_inputs(q, k, v, layout)
    shape, dtype, dev = q.shape, q.dtype, q.device
    if do.shape != shape or do.dtype != dtype or do.device != dev:
        raise ValueError("do must be a bfloat16 tensor shaped like q on its device")
    if o.shape != shape or o.dtype != dtype or o.device != dev:
        raise ValueError("o must be a bfloat16 tensor shaped like q on its device")
    batch, heads, sq, d = shape[0], shape[hd], shape[sd], shape[3]
    heads_kv, skv = k.shape[hd], k.shape[sd]
    if lse.shape != (batch, heads, sq) or lse.dtype != torch.float32 or lse.device != dev:
        raise ValueError("lse must be float32 [batch, heads, seq_len] on the device of q")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(d)
    do, q, k, v, o, lse = (_lib.aligned(do), _lib.aligned(q), _lib.aligned(k), _lib.aligned(v), _lib.aligned(o),
                           _lib.aligned(lse))
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    causal = 1 if causal else 0
    need = _workspace_bytes(batch, heads, heads_kv, sq, skv, d, causal, dev) if batch and sq else 0
    # from the allocator on every call: calls on several streams and captured graphs do not share it
    workspace = _lib.empty((need or 1,), torch.uint8, dev)
    status = _lib.host_status_ptr(dev, "flash_attention_2_bwd")
    rc = _lib.call_on(dev, _lib.load().tokmix_fa2_bwd, do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                      lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), batch, heads, heads_kv, sq, skv, d,
                      _lib.LAYOUT_BHSD if layout == "bhsd" else _lib.LAYOUT_BSHD, causal, float(sm_scale),
                      workspace.data_ptr(), need, status, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "flash_attention_2_bwd")
    _lib.after_host_status_launch(dev, "flash_attention_2_bwd")
    return dq, dk, dv


def check_device_status(device: torch.device | None = None) -> None:
    """Synchronise and raise if a call on `device` reported a device-side timeout."""
    dev = torch.device(device) if device is not None else torch.device("cuda")
    dev = torch.device("cuda", dev.index if dev.index is not None else torch.cuda.current_device())
    torch.cuda.synchronize(dev)
    _lib.take_host_status(dev, "flash_attention_2_bwd")


def get_inputs(batch: int = 8, head_num: int = 8, seq_len: int = 2048, head_dim: int = 128,
               dtype: torch.dtype = torch.bfloat16, causal: bool = True, seed: int = 42, *,
               head_num_kv: int | None = None, layout: str = "bhsd", device: str = "cuda") -> dict:
    """The forward's inputs and its outputs, and an N(0,1) gradient of the output."""
    inp = _forward.get_inputs(batch, head_num, seq_len, head_dim, dtype, causal, seed, head_num_kv=head_num_kv,
                              layout=layout, device=device)
    inp["o"], inp["lse"] = _forward.kernel_fn(**inp, return_lse=True)
    gen = torch.Generator().manual_seed(seed + 1)
    inp["do"] = torch.randn(inp["q"].shape, generator=gen).to(dtype).to(device)
    return inp


def get_flops(batch: int = 8, head_num: int = 8, seq_len: int = 2048, head_dim: int = 128, causal: bool = True) -> int:
    """Five products over the visible pairs (the forward has two)."""
    return _forward.get_flops(batch, head_num, seq_len, head_dim, causal) * 5 // 2


def get_bytes(batch: int = 8, head_num: int = 8, seq_len: int = 2048, head_dim: int = 128, element_size: int = 2, *,
              head_num_kv: int | None = None) -> int:
    """q, k, v, o, do and lse read once, dq, dk and dv written once."""
    hkv = head_num if head_num_kv is None else head_num_kv
    return batch * seq_len * (4 * (head_num + hkv) * head_dim * element_size + 4 * head_num)
