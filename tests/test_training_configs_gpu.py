"""The training operators at their configs' sizes, through the harness's own checkers and tolerances."""

import pytest
import torch

from kernel_opt_agent_b200 import flash_attention_2_bwd, qk_norm_rope, qk_norm_rope_bwd
from kernel_opt_agent_b200.kernel_configs import KERNEL_CONFIGS

pytestmark = pytest.mark.gpu
MODULES = {"qk_norm_rope": qk_norm_rope, "qk_norm_rope_bwd": qk_norm_rope_bwd, "flash_attention_2_bwd": flash_attention_2_bwd}
CASES = [(name, label, size, dt) for name in MODULES for label, size in KERNEL_CONFIGS[name]["test_sizes"] + KERNEL_CONFIGS[name][
    "edge_sizes"] for dt in KERNEL_CONFIGS[name]["test_dtypes"]]


@pytest.mark.parametrize("name,label,size,dtype", CASES, ids=[f"{n}-{lb}-{str(d)[6:]}" for n, lb, _, d in CASES])
def test_config_sizes(cuda_device, name, label, size, dtype):
    cfg, mod = KERNEL_CONFIGS[name], MODULES[name]
    assert mod.KERNEL_TYPE == name
    inp = cfg["input_generator"](size, dtype, "cuda")
    got, ref = mod.kernel_fn(**inp), cfg["reference_fn"](inp)
    assert len(got) == len(ref)
    for x, r in zip(got, ref):
        assert x.shape == r.shape and x.dtype == r.dtype
        torch.testing.assert_close(x.float(), r.float(), **cfg["tolerances"][dtype])
    assert cfg["flops_fn"](size) > 0 and cfg["bytes_fn"](size, dtype) > 0
    mod.check_device_status(cuda_device)


@pytest.mark.parametrize("name", MODULES)
def test_module_inputs_run(cuda_device, name):
    mod = MODULES[name]
    inp = mod.get_inputs(seq_len=64, batch=1) if name != "flash_attention_2_bwd" else mod.get_inputs(1, 4, 64, 64)
    assert all(torch.isfinite(t.float()).all() for t in mod.kernel_fn(**inp))
    assert mod.get_flops() > 0 and mod.get_bytes() > 0
