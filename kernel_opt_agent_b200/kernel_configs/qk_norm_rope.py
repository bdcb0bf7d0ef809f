"""qk_norm_rope config callables: slices of a packed N(0,1) projection of scale 2, weights about 1, rotary tables in
fp32, from a seeded CPU generator; ``axes`` > 1 gives random positions with that many axes, their shares of the pairs equal (the
first takes what is left) and dealt out in turn.  The checker is ``references.qk_norm_rope_ref``."""

from __future__ import annotations

import torch

from kernel_opt_agent_b200 import references
from ._utils import dtype_bytes

KERNEL_OPT_CHARACTERISTICS = {
    "is_matmul_like": False,
    "supports_tensor_core_candidate": False,
    "memory_bound": True,
}


def input_generator(size: dict, dtype: torch.dtype, device: str, seed: int = 42) -> dict:
    from kernel_opt_agent_b200.qk_norm_rope import get_inputs
    b, s, pairs, axes = (int(size[n]) for n in ("batch", "seq_len", "pairs", "axes"))
    inp = get_inputs(b, s, int(size["q_heads"]), int(size["kv_heads"]), int(size["head_dim"]), pairs, dtype, seed, device)
    inp["nope_dim"] = int(size["nope_dim"])
    if axes > 1:
        gen = torch.Generator().manual_seed(seed + 2)
        inp["positions"] = torch.randint(0, s, (axes, b, s), generator=gen).int().to(device)
        share = pairs // axes
        inp["sections"], inp["interleaved"] = (pairs - share * (axes - 1),) + (share,) * (axes - 1), True
    return inp


def reference_fn(inputs: dict):
    return references.qk_norm_rope_ref(**inputs)


def _elements(size: dict) -> int:
    return (int(size["batch"]) * int(size["seq_len"]) * (int(size["q_heads"]) + int(size["kv_heads"]))
            * int(size["head_dim"]))


def flops_fn(size: dict) -> int:
    return 8 * _elements(size)


def bytes_fn(size: dict, dtype: torch.dtype) -> int:
    """q and k read and written once, the tables' rows and the positions read once, the weights."""
    s, axes = int(size["seq_len"]), int(size["axes"])
    positions = axes * int(size["batch"]) * s * 4 if axes > 1 else 0
    return _elements(size) * dtype_bytes(dtype) * 2 + s * int(size["pairs"]) * 8 + positions + 2 * int(
        size["head_dim"]) * dtype_bytes(dtype)
