"""add_rms_norm_quant config callables: N(0,1) x, a residual stream of 4 N(0,1) and weights about 1 from a seeded
CPU generator; the checker is ``references.add_rms_norm_quant_ref``."""

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
    gen = torch.Generator().manual_seed(seed)
    m, n = int(size["M"]), int(size["N"])
    return {"x": torch.randn(m, n, generator=gen).to(dtype).to(device),
            "residual": (4 * torch.randn(m, n, generator=gen)).to(dtype).to(device),
            "weight": (1 + 0.2 * torch.randn(n, generator=gen)).to(dtype).to(device),
            "group": int(size["group"]) or None}


def reference_fn(inputs: dict):
    return references.add_rms_norm_quant_ref(**inputs)


def flops_fn(size: dict) -> int:
    return 7 * int(size["M"]) * int(size["N"])


def bytes_fn(size: dict, dtype: torch.dtype) -> int:
    """x and residual read, their sum and the e4m3 row written, the fp32 scales, the weight read once."""
    m, n = int(size["M"]), int(size["N"])
    eb = dtype_bytes(dtype)
    return m * n * (3 * eb + 1) + n * eb + m * (n // int(size["group"]) if size["group"] else 1) * 4
