"""qk_norm_rope and its gradient with eps = 0, and for rows at the ends of the range of their squares, against the formulas in
64 bits (the bounds of test_qk_norm_rope_gpu.py)."""

import pytest
import torch

from kernel_opt_agent_b200 import qk_norm_rope as norm
from kernel_opt_agent_b200 import qk_norm_rope_bwd as bwd
from tests.test_qk_norm_rope_gpu import BF16, FP16, FP32, close, formula, formula_bwd, make, turns

pytestmark = pytest.mark.gpu


def check(q, k, qw, kw, cos, sin, pos, dy, eps, nope=0, slack=0.0):
    """slack: what the inverse root may be off besides, of itself."""
    c, sn = turns(cos, sin, pos, q.shape[0], q.shape[1], None, False)
    d = q.shape[-1]
    more = 1 + slack * 2.0 ** 24 / (d / 2 + 16)      # the bounds are (d / 2 + 16) 2^-24 of the absolute sums, or more
    for y, x, w in zip(norm.kernel_fn(q, k, qw, kw, cos, sin, pos, eps=eps, nope_dim=nope), (q, k), (qw, kw)):
        ref, err = formula(x, w, c, sn, nope, eps)
        close(y, ref, err * more)
    dq, dk, dqw, dkw = bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin, pos, eps=eps, nope_dim=nope)
    for dx, dw, g, x, w in ((dq, dqw, dy[0], q, qw), (dk, dkw, dy[1], k, kw)):
        assert torch.isfinite(dw).all()
        ref, err, wref, werr = formula_bwd(g, x, w, c, sn, nope, eps)
        close(dx, ref, err * more)
        close(dw, wref, werr * more)
    norm.check_device_status(q.device)


@pytest.mark.parametrize("b,s,hq,hk,d,dtype,wtype", [
    (1, 1, 3, 1, 64, BF16, None), (2, 37, 5, 3, 64, BF16, FP32), (1, 300, 1, 2, 64, FP16, None), (2, 9, 5, 1, 128, BF16, None),
    (1, 129, 3, 3, 128, FP16, FP32), (2, 21, 3, 1, 256, BF16, FP32), (1, 40, 8, 4, 64, BF16, None)])
def test_without_eps(cuda_device, b, s, hq, hk, d, dtype, wtype):
    """Head counts that do not fill the last iteration of 256 / D heads, and some that do."""
    check(*make(b, s, hq, hk, d, d // 4, dtype, wtype, far=s + 50, seed=s + d), eps=0.0)


@pytest.mark.parametrize("power", [-66, -62, 59])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_at_the_ends_of_the_range(cuda_device, power, d):
    """Rows of magnitude 2^power, whose inverse root lies at the other end of fp32's range.  At 2^-66 squares and their mean are
    below fp32's normal numbers: each of the d squares, their sums and the mean are off by at most 2^-150, so the mean, 2^-132, by
    2^-17 of itself, the inverse root by half of that, and dx, which has it three times, by less than 2^-16."""
    q, k, qw, kw, cos, sin, pos, dy = make(2, 19, 3, 1, d, 16, BF16, FP32, seed=d, packed=False)
    q, k = ((x / x.float().square().mean(-1, keepdim=True).sqrt() * 2.0 ** power).to(BF16) for x in (q, k))
    check(q, k, qw, kw, cos, sin, pos, dy, eps=0.0, slack=2.0 ** -16 if power < -63 else 0.0)


def test_a_zero_row_without_eps(cuda_device):
    """0 / 0 as the formula has it: NaN in the row and in its kind's weight gradient, nowhere else."""
    q, k, qw, kw, cos, sin, pos, dy = make(2, 5, 3, 1, 64, 8, FP16, FP32, packed=False)
    want, want_g = norm.kernel_fn(q, k, qw, kw, cos, sin, eps=0.0), bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin, eps=0.0)
    q[1, 2, 2] = 0
    got, grads = norm.kernel_fn(q, k, qw, kw, cos, sin, eps=0.0), bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin, eps=0.0)
    keep = torch.ones(2, 5, 3, dtype=torch.bool, device=q.device)
    keep[1, 2, 2] = False
    for y, ref in ((got[0], want[0]), (grads[0], want_g[0])):
        assert torch.equal(y[keep], ref[keep]) and y[~keep].isnan().all()
    assert torch.equal(got[1], want[1]) and torch.equal(grads[1], want_g[1]) and torch.equal(grads[3], want_g[3])
    assert torch.isfinite(grads[3]).all() and grads[2].isnan().all()
