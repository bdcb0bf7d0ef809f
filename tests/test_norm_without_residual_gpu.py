"""add_rms_norm_quant without a residual returns the very x it was given, read in place or not."""

import pytest
import torch

from kernel_opt_agent_b200 import add_rms_norm_quant as norm
from kernel_opt_agent_b200 import references

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [None, 32, 128])
def test_the_residual_of_the_first_layer_is_x(cuda_device, group):
    gen = torch.Generator().manual_seed(3)
    flat = torch.randn(2 * 5 * 300, generator=gen).to(torch.bfloat16).to(cuda_device)
    weight = torch.randn(256, generator=gen).to(torch.bfloat16).to(cuda_device)
    for x in (flat[:1280].view(5, 256), flat[1:1281].view(5, 256), flat.view(2, 5, 300)[:, :, :256], flat[:512].view(256, 2).t()):
        y, scale, h = norm.kernel_fn(x, None, weight, group=group)
        assert h is x
        want_y, want_scale, _ = references.add_rms_norm_quant_ref(x.contiguous(), None, weight, group=group)
        assert y.shape == x.shape and torch.equal(y.contiguous().view(torch.uint8), want_y.view(torch.uint8))
        torch.testing.assert_close(scale, want_scale, rtol=1e-5, atol=0)
