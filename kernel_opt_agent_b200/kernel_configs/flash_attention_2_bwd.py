"""flash_attention_2_bwd config callables: flash_attention_2's inputs, its output and log-sum-exp, and an N(0,1) gradient;
the checker is ``references.flash_attention_2_bwd_ref``."""

from __future__ import annotations

import torch

from kernel_opt_agent_b200 import references
from . import flash_attention_2 as _forward

KERNEL_OPT_CHARACTERISTICS = _forward.KERNEL_OPT_CHARACTERISTICS


def input_generator(size: dict, dtype: torch.dtype, device: str, seed: int = 42) -> dict:
    from kernel_opt_agent_b200 import flash_attention_2
    inp = _forward.input_generator(size, dtype, device, seed)
    inp["o"], inp["lse"] = flash_attention_2.kernel_fn(**inp, return_lse=True)
    gen = torch.Generator().manual_seed(seed + 1)
    inp["do"] = torch.randn(inp["q"].shape, generator=gen).to(dtype).to(device)
    return inp


def reference_fn(inputs: dict):
    return references.flash_attention_2_bwd_ref(**inputs)


def flops_fn(size: dict) -> int:
    """Five products over the visible pairs where the forward has two."""
    return _forward.flops_fn(size) * 5 // 2


def bytes_fn(size: dict, dtype: torch.dtype) -> int:
    """q, k, v, o and do read, dq, dk and dv written, lse read."""
    lse = 4 * size["batch"] * size["head_num"] * size["seq_len"]
    return 2 * _forward.bytes_fn(size, dtype) + lse
