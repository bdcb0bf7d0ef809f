"""kv8_append config callables: N(0,1) new tokens behind a cache of zeros at scale 2^-8 (the module's get_inputs);
the checker is ``references.kv8_append_ref``, which copies the cache (the kernel updates it, and appending the
same tokens at the same positions again changes nothing)."""

from __future__ import annotations

import torch

from kernel_opt_agent_b200 import kv8_append, references
from ._utils import dtype_bytes

KERNEL_OPT_CHARACTERISTICS = {
    "is_matmul_like": False,
    "supports_tensor_core_candidate": False,
    "memory_bound": True,
}


def input_generator(size: dict, dtype: torch.dtype, device: str, seed: int = 42) -> dict:
    params = dict(size)
    params["cache_dtype"] = getattr(torch, size["cache_dtype"])
    return kv8_append.get_inputs(**params, dtype=dtype, seed=seed, device=device)


def reference_fn(inputs: dict):
    return references.kv8_append_ref(**inputs)


def flops_fn(size: dict) -> int:
    return kv8_append.get_flops(size["batch"], size["tokens"], size["head_num_kv"], size["head_dim"])


def bytes_fn(size: dict, dtype: torch.dtype) -> int:
    return kv8_append.get_bytes(size["batch"], size["tokens"], size["head_num_kv"], size["head_dim"],
                                dtype_bytes(dtype))
