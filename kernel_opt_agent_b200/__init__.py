"""B200-native (sm_100a) prefill token mixers behind the kernel_opt_agent plugin contract.

Plugin modules (drop-ins for the reference's ``kernels_optimized/<name>.py``):
  * :mod:`kernel_opt_agent_b200.flash_attention_2`     -- causal attention forward
  * :mod:`kernel_opt_agent_b200.qwen35moe_gdn_prefill` -- chunked gated-delta-rule prefill

Beside them, the serving step's operators, modules of the same contract:
  * :mod:`kernel_opt_agent_b200.add_rms_norm_quant` -- residual addition, RMS norm, FP8 output
  * :mod:`kernel_opt_agent_b200.kv8_append`         -- new keys/values into a paged 8-bit cache
  * :mod:`kernel_opt_agent_b200.kv8_attention`      -- decode attention over that cache

And training the attention layers:
  * :mod:`kernel_opt_agent_b200.qk_norm_rope`          -- norm of each query and key head with the position rotation
  * :mod:`kernel_opt_agent_b200.qk_norm_rope_bwd`      -- its gradient
  * :mod:`kernel_opt_agent_b200.flash_attention_2_bwd` -- the attention's gradient
  * :mod:`kernel_opt_agent_b200.training`              -- the same behind autograd

All call the hand-written kernels in ``libtokmix.so`` (the prefill mixers and the attention's gradient on tcgen05 and TMA, the serving step on
``mma.sync``, ``cp.async`` and plain loads) through the C ABI in ``include/tokmix.h``.  ``kernel_configs`` and ``references`` mirror the reference's registry and
checkers; ``sharding`` holds the multi-GPU work partition.
"""

from . import (add_rms_norm_quant, flash_attention_2, flash_attention_2_bwd, kv8_append, kv8_attention,  # noqa: F401
               qk_norm_rope, qk_norm_rope_bwd, qwen35moe_gdn_prefill, training)

__all__ = ["add_rms_norm_quant", "flash_attention_2", "flash_attention_2_bwd", "kv8_append", "kv8_attention",
           "qk_norm_rope", "qk_norm_rope_bwd", "qwen35moe_gdn_prefill", "training"]
