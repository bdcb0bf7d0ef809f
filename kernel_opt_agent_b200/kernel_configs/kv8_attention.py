"""kv8_attention config callables: N(0,1) queries, keys and values (the module's get_inputs); the checker is
``references.kv8_attention_ref``."""

from __future__ import annotations

import torch

from kernel_opt_agent_b200 import kv8_attention, references
from ._utils import dtype_bytes

KERNEL_OPT_CHARACTERISTICS = {
    "is_matmul_like": True,
    "supports_tensor_core_candidate": True,
    "memory_bound": True,
}


def input_generator(size: dict, dtype: torch.dtype, device: str, seed: int = 42) -> dict:
    params = dict(size)
    params["cache_dtype"] = getattr(torch, size["cache_dtype"])
    return kv8_attention.get_inputs(**params, dtype=dtype, seed=seed, device=device)


def reference_fn(inputs: dict) -> torch.Tensor:
    return references.kv8_attention_ref(**inputs)


def flops_fn(size: dict) -> int:
    return kv8_attention.get_flops(size["batch"], size["tokens"], size["seq_len"], size["head_num"], size["head_dim"])


def bytes_fn(size: dict, dtype: torch.dtype) -> int:
    return kv8_attention.get_bytes(size["batch"], size["tokens"], size["seq_len"], size["head_num"],
                                   size["head_num_kv"], size["head_dim"], dtype_bytes(dtype))
