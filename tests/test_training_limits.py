"""Arguments beyond what the training operators can hold are refused before anything is launched (CPU only)."""

import pytest
import torch

from kernel_opt_agent_b200 import qk_norm_rope, qk_norm_rope_bwd


@pytest.mark.parametrize("eps", [1e39, 1e300, float("inf"), float("nan"), -1e-9, -float("inf")])
def test_eps_that_fp32_cannot_hold(eps):
    q, w, t = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16), torch.zeros(64), torch.zeros(2, 8)
    with pytest.raises(ValueError, match="eps"):
        qk_norm_rope.kernel_fn(q, q, w, w, t, t, eps=eps)
    with pytest.raises(ValueError, match="eps"):
        qk_norm_rope_bwd.kernel_fn(q, q, q, q, w, w, t, t, eps=eps)
