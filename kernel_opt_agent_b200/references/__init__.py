"""Correctness references for the harness (mirror of the reference's ``references/``).

These are the checkers ``kernel_configs/*.reference_fn`` call, as in the reference
(``references/__init__.py:7-23``).  They are plain PyTorch on the inputs' device and never part
of a kernel_fn call.
"""

from .add_rms_norm_quant import add_rms_norm_quant_ref
from .flash_attention_2 import flash_attention_2_ref
from .kv8 import kv8_append_ref, kv8_attention_ref, kv8_values
from .qkv_part_rope import qkv_part_rope_ref
from .qwen35moe_gdn_prefill import qwen35moe_gdn_prefill_ref
from .rms_norm import rms_norm_ref
from .swiglu_input_quant import swiglu_input_quant_ref

__all__ = ["add_rms_norm_quant_ref", "flash_attention_2_ref", "kv8_append_ref", "kv8_attention_ref", "kv8_values",
           "qkv_part_rope_ref", "qwen35moe_gdn_prefill_ref", "rms_norm_ref", "swiglu_input_quant_ref"]
