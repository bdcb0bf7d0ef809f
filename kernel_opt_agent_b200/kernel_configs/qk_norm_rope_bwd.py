"""qk_norm_rope_bwd config callables: qk_norm_rope's inputs and N(0,1) gradients of its outputs; the checker is
``references.qk_norm_rope_bwd_ref``."""

from __future__ import annotations

import torch

from kernel_opt_agent_b200 import references
from . import qk_norm_rope as _forward
from ._utils import dtype_bytes

KERNEL_OPT_CHARACTERISTICS = _forward.KERNEL_OPT_CHARACTERISTICS


def input_generator(size: dict, dtype: torch.dtype, device: str, seed: int = 42) -> dict:
    inp = _forward.input_generator(size, dtype, device, seed)
    gen = torch.Generator().manual_seed(seed + 1)
    return {"dq_out": torch.randn(inp["q"].shape, generator=gen).to(dtype).to(device),
            "dk_out": torch.randn(inp["k"].shape, generator=gen).to(dtype).to(device), **inp}


def reference_fn(inputs: dict):
    return references.qk_norm_rope_bwd_ref(**inputs)


def flops_fn(size: dict) -> int:
    return 2 * _forward.flops_fn(size)


def bytes_fn(size: dict, dtype: torch.dtype) -> int:
    """As the forward, with the gradients of the outputs read beside q and k."""
    return _forward.bytes_fn(size, dtype) + (_forward._elements(size) + 2 * int(size["head_dim"])) * dtype_bytes(dtype)
