"""The head norm with rotation and its gradient on a B200 against the formulas in 64 bits.

Tolerances.  The kernels compute in fp32 (2^-24 a rounding) and round once to the output's type (at most half a step,
eps / 2 of the value).  Forward: y is a sum of two products x * (r w cos); r has the sum of D squares (D + 8
roundings at the worst, halved by the root) and the root's own error behind it, each product four roundings more, so
each term is off by less than (D / 2 + 16) 2^-24 of itself.  Backward: the same for g and for the mean of D products, twice
over; the weights' gradients are sums of n rows, off by at most n 2^-24 of their absolute sum.  The absolute sums are
formed in 64 bits beside the formula.
"""

import pytest
import torch

from kernel_opt_agent_b200 import _lib, training
from kernel_opt_agent_b200 import qk_norm_rope as norm
from kernel_opt_agent_b200 import qk_norm_rope_bwd as bwd

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TINY = {BF16: 2.0 ** -133, FP16: 2.0 ** -25, FP32: 2.0 ** -149}  # half the smallest step


def axis_of_pairs(half, sections, interleaved):
    if sections is None:
        return [0] * half
    if interleaved:
        a = len(sections)
        return [j % a if j < a * sections[j % a] else 0 for j in range(half)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


def turns(cos, sin, positions, b, s, sections, interleaved):
    """cos and sin of every token's pairs, float64 [B, S, 1, half]."""
    half = cos.shape[1]
    if positions is None:
        positions = torch.arange(s, device=cos.device).expand(b, s)
    pos = positions.long() if positions.ndim == 3 else positions.long()[None]
    axis = torch.tensor(axis_of_pairs(half, sections, interleaved), device=cos.device)
    rows = pos[axis].permute(1, 2, 0)
    pair = torch.arange(half, device=cos.device)
    return cos.double()[rows, pair][:, :, None], sin.double()[rows, pair][:, :, None]


def rotate(n, c, s, nope):
    half = c.shape[-1]
    a, b = n[..., nope:nope + half], n[..., nope + half:nope + 2 * half]
    return torch.cat((n[..., :nope], a * c - b * s, a * s + b * c, n[..., nope + 2 * half:]), -1)


def formula(x, w, c, s, nope, eps):
    """The forward of one kind of heads in float64 and the bound of its fp32 error."""
    x, w = x.double(), w.double()
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    err = rotate(n.abs(), c.abs(), -s.abs(), nope)
    err[..., nope + c.shape[-1]:nope + 2 * c.shape[-1]] = rotate(n.abs(), c.abs(), s.abs(), nope)[
        ..., nope + c.shape[-1]:nope + 2 * c.shape[-1]]
    return rotate(n, c, s, nope), err * (x.shape[-1] / 2 + 16) * 2.0 ** -24


def formula_bwd(dy, x, w, c, s, nope, eps):
    """(dx, dw) in float64 and the bounds of their fp32 errors."""
    dy, x, w = dy.double(), x.double(), w.double()
    d, half = x.shape[-1], c.shape[-1]
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    g = rotate(dy, c, -s, nope)
    ga = rotate(dy.abs(), c.abs(), -s.abs(), nope)
    ga[..., nope + half:nope + 2 * half] = rotate(dy.abs(), c.abs(), s.abs(), nope)[..., nope + half:nope + 2 * half]
    dx = r * (g * w - x * r * r * (g * w * x).mean(-1, keepdim=True))
    dx_abs = r * (ga * w.abs() + x.abs() * r * r * (ga * (w * x).abs()).mean(-1, keepdim=True))
    dw, dw_abs = (g * x * r).sum((0, 1, 2)), (ga * x.abs() * r).sum((0, 1, 2))
    rows = x[..., 0].numel()
    return dx, dx_abs * (2 * d + 32) * 2.0 ** -24, dw, dw_abs * (d / 2 + 32 + rows) * 2.0 ** -24


def close(got, ref, err):
    t = got.dtype
    bound = err + ref.abs() * torch.finfo(t).eps / 2 * (1 + 2.0 ** -20) + TINY[t]
    used = ((got.double() - ref).abs() / bound).max().item() if ref.numel() else 0.0
    assert used <= 1.0, used


def make(b, s, hq, hk, d, half, dtype, wtype, sections=None, far=0, seed=0, packed=True, order=None):
    gen = torch.Generator().manual_seed(seed)
    heads = hq + 2 * hk
    qkv = (torch.randn(b, s, heads, d, generator=gen) * torch.exp2(torch.randn(heads, 1, generator=gen))).to(dtype).cuda()
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    if not packed:
        q, k = q.contiguous(), k.contiguous()
    rows = max(far, s) + 3
    cos, sin = norm.rotary_tables(rows, half)
    pos = None
    if sections is not None:
        pos = torch.randint(0, rows, (len(sections), b, s), generator=gen).int().cuda()
    elif far:
        pos = torch.randint(0, rows, (b, s), generator=gen).int().cuda()
    w = [(1 + 0.3 * torch.randn(d, generator=gen)).to(wtype or dtype).cuda() for _ in range(2)]
    dy = [torch.randn(b, s, h, d, generator=gen).to(dtype).cuda() for h in (hq, hk)]
    return q, k, w[0], w[1], cos, sin, pos, dy


CASES = [
    # b, s, hq, hk, d, half, nope, dtype, weights, sections, interleaved, far
    (1, 1, 1, 1, 64, 8, 0, BF16, None, None, False, 0),
    (1, 1, 16, 2, 256, 32, 192, BF16, None, None, False, 70000),
    (64, 1, 10, 1, 256, 32, 0, FP16, FP32, None, False, 1000),
    (2, 333, 4, 2, 128, 64, 0, BF16, None, None, False, 0),
    (3, 17, 3, 1, 64, 32, 0, FP16, None, None, False, 99),
    (1, 129, 5, 3, 64, 16, 16, BF16, FP32, None, False, 0),
    (2, 31, 7, 1, 128, 24, 40, FP16, None, None, False, 50),
    (1, 65, 8, 8, 256, 128, 0, BF16, FP32, None, False, 0),
    (2, 50, 8, 2, 128, 64, 0, BF16, None, (16, 24, 24), False, 0),
    (2, 50, 8, 2, 128, 64, 0, FP16, None, (24, 20, 20), True, 0),
    (1, 70, 2, 1, 256, 32, 64, BF16, FP32, (11, 11, 10), True, 0),
    (1, 9, 3, 2, 64, 16, 32, BF16, None, (4, 4, 4, 4), False, 0),
    (2, 9, 3, 2, 64, 24, 8, FP16, None, (20, 4), True, 0),
    (1, 20, 4, 1, 128, 16, 96, BF16, None, (16, 0), False, 0),
    (1, 20, 4, 1, 128, 16, 96, BF16, None, (16,), False, 0),
    (1, 5000, 2, 1, 128, 64, 0, BF16, FP32, None, False, 0),   # enough tokens for one warp each
    (2, 4099, 5, 2, 64, 32, 0, FP16, None, None, False, 0),
]


@pytest.mark.parametrize("b,s,hq,hk,d,half,nope,dtype,wtype,sections,inter,far", CASES)
@pytest.mark.parametrize("packed", [True, False])
def test_matches_the_formula(cuda_device, b, s, hq, hk, d, half, nope, dtype, wtype, sections, inter, far, packed):
    q, k, qw, kw, cos, sin, pos, dy = make(b, s, hq, hk, d, half, dtype, wtype, sections, far, seed=s + d + hq, packed=packed)
    kw_args = dict(eps=1e-6, nope_dim=nope, sections=sections, interleaved=inter)
    c, sn = turns(cos, sin, pos, b, s, sections, inter)
    got = norm.kernel_fn(q, k, qw, kw, cos, sin, pos, **kw_args)
    for y, x, w in zip(got, (q, k), (qw, kw)):
        assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
        close(y, *formula(x, w, c, sn, nope, 1e-6))
    dq, dk, dqw, dkw = bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin, pos, **kw_args)
    for dx, dw, g, x, w in ((dq, dqw, dy[0], q, qw), (dk, dkw, dy[1], k, kw)):
        assert dx.shape == x.shape and dx.dtype == dtype and dx.is_contiguous() and dw.dtype == w.dtype
        ref, err, wref, werr = formula_bwd(g, x, w, c, sn, nope, 1e-6)
        close(dx, ref, err)
        close(dw, wref, werr)
    norm.check_device_status(cuda_device)


def test_gradient_against_differences(cuda_device):
    """The formula that the kernel is tested against is the forward's derivative (float64, central differences)."""
    q, k, qw, kw, cos, sin, pos, dy = make(1, 3, 2, 1, 64, 16, BF16, FP32, seed=5)
    c, sn = turns(cos, sin, pos, 1, 3, None, False)
    x, w, g = q.double(), qw.double(), dy[0].double()
    dx, _, dw, _ = formula_bwd(g, x, w, c, sn, 32, 1e-6)
    f = lambda x, w: (formula(x, w, c, sn, 32, 1e-6)[0] * g).sum()  # noqa: E731
    h = 2.0 ** -16
    for at in [(0, 0, 0, 0), (0, 1, 1, 33), (0, 2, 0, 63), (0, 2, 1, 50)]:
        step = torch.zeros_like(x)
        step[at] = h
        assert abs((f(x + step, w) - f(x - step, w)) / (2 * h) - dx[at]).item() < 1e-6
    for at in (0, 31, 32, 63):
        step = torch.zeros_like(w)
        step[at] = h
        assert abs((f(x, w + step) - f(x, w - step)) / (2 * h) - dw[at]).item() < 1e-6


def test_default_rotation_is_the_last_columns(cuda_device):
    q, k, qw, kw, cos, sin, _, _ = make(1, 12, 2, 1, 128, 16, BF16, None)
    a = norm.kernel_fn(q, k, qw, kw, cos, sin)
    b = norm.kernel_fn(q, k, qw, kw, cos, sin, nope_dim=96)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_values_that_are_not_finite_stay_in_their_rows(cuda_device):
    q, k, qw, kw, cos, sin, _, dy = make(1, 40, 4, 2, 128, 32, BF16, None, seed=3, packed=False)
    want = norm.kernel_fn(q, k, qw, kw, cos, sin)
    want_g = bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin)
    q[0, 7, 1, 5], q[0, 8, 2, 100], k[0, 9, 0, 0] = float("nan"), float("inf"), float("-inf")
    got = norm.kernel_fn(q, k, qw, kw, cos, sin)
    grads = bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin)
    for y, ref, bad in ((got[0], want[0], [(7, 1), (8, 2)]), (got[1], want[1], [(9, 0)]),
                        (grads[0], want_g[0], [(7, 1), (8, 2)]), (grads[1], want_g[1], [(9, 0)])):
        keep = torch.ones(y.shape[:3], dtype=torch.bool, device=y.device)
        for t, h in bad:
            keep[0, t, h] = False
        assert torch.equal(y[keep], ref[keep])
    assert got[0][0, 7, 1].isnan().all() and grads[0][0, 7, 1].isnan().all() and grads[2].isnan().all()
    # one infinite value: its row's inverse root is 0, the row 0 but for 0 * inf in the value's own pair
    row = got[0][0, 8, 2]
    assert row[100].isnan() and row[:64].eq(0).all()


def test_zero_rows(cuda_device):
    q, k, qw, kw, cos, sin, _, dy = make(2, 5, 3, 1, 64, 8, FP16, FP32, packed=False)
    q[0, 2] = 0
    y, _ = norm.kernel_fn(q, k, qw, kw, cos, sin)
    assert (y[0, 2] == 0).all() and torch.isfinite(y).all()
    dq, _, dqw, _ = bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin, eps=1e-2)
    c, sn = turns(cos, sin, None, 2, 5, None, False)
    ref, err, wref, werr = formula_bwd(dy[0], q, qw, c, sn, 48, 1e-2)
    close(dq, ref, err)
    close(dqw, wref, werr)


@pytest.mark.parametrize("b,s", [(0, 5), (3, 0), (0, 0)])
def test_empty(cuda_device, b, s):
    q, k, qw, kw, cos, sin, _, dy = make(b, s, 3, 1, 64, 8, BF16, None)
    y = norm.kernel_fn(q, k, qw, kw, cos, sin)
    assert y[0].shape == (b, s, 3, 64) and y[1].shape == (b, s, 1, 64)
    g = bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin)
    assert g[0].shape == q.shape and g[2].eq(0).all() and g[3].eq(0).all()


def test_views_and_broadcast_gradients(cuda_device):
    """Heads before tokens, every second head, gradients that are expanded or transposed, odd addresses."""
    q, k, qw, kw, cos, sin, _, dy = make(2, 37, 4, 2, 128, 64, BF16, None, seed=8, packed=False)
    want = norm.kernel_fn(q, k, qw, kw, cos, sin)
    want_g = bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin)
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(2, 37, 4, 128, dtype=BF16, device=q.device)
    wide[:, :, ::2] = k
    odd = torch.zeros(q.numel() + 3, dtype=BF16, device=q.device)[3:].view(q.shape).copy_(q)
    for qq, kk in ((qt, wide[:, :, ::2]), (odd, k)):
        got = norm.kernel_fn(qq, kk, qw, kw, cos, sin)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        dyt = [g.transpose(1, 2).contiguous().transpose(1, 2) for g in dy]
        grads = bwd.kernel_fn(*dyt, qq, kk, qw, kw, cos, sin)
        assert all(torch.equal(x, y) for x, y in zip(grads, want_g))
    one = torch.ones((), dtype=BF16, device=q.device)
    a = bwd.kernel_fn(one.expand(q.shape), one.expand(k.shape), q, k, qw, kw, cos, sin)
    b = bwd.kernel_fn(torch.ones_like(q), torch.ones_like(k), q, k, qw, kw, cos, sin)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_same_bits_every_time(cuda_device):
    q, k, qw, kw, cos, sin, _, dy = make(2, 3001, 6, 2, 128, 64, BF16, FP32, seed=2)
    first = bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin)))


@pytest.mark.parametrize("sections", [None, (16, 24, 24)])
def test_positions_outside_the_tables(cuda_device, sections):
    q, k, qw, kw, cos, sin, pos, dy = make(2, 9, 3, 1, 128, 64, BF16, None, sections=sections, far=20, seed=6)
    rows = cos.shape[0]
    want = norm.kernel_fn(q, k, qw, kw, cos, sin, pos, sections=sections)
    bad = pos.clone()
    flat = bad if bad.ndim == 2 else bad[1]
    flat[0, 3], flat[1, 8], flat[1, 2] = rows, -1, 2 ** 31 - 1
    got = norm.kernel_fn(q, k, qw, kw, cos, sin, bad, sections=sections)
    with pytest.raises(_lib.TokmixDeviceError):
        norm.check_device_status(cuda_device)
    keep = torch.ones(2, 9, dtype=torch.bool, device=q.device)
    keep[0, 3] = keep[1, 8] = keep[1, 2] = False
    for y, ref in zip(got, want):
        assert torch.equal(y[keep], ref[keep]) and y[~keep].isnan().all()
    grads = bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin, bad, sections=sections)
    with pytest.raises(_lib.TokmixDeviceError):
        bwd.check_device_status(cuda_device)
    assert torch.isfinite(grads[0][keep]).all() and grads[0][~keep].isnan().all()
    norm.check_device_status(cuda_device)


def test_captured_and_replayed(cuda_device):
    """A graph's replays follow its inputs, and two graphs do not share the weights' partial sums."""
    state = [make(2, 200, 4, 2, 64, 32, BF16, FP32, far=500, seed=i, packed=False) for i in range(4)]

    def step(t):
        q, k, qw, kw, cos, sin, pos, dy = t
        return [*norm.kernel_fn(q, k, qw, kw, cos, sin, pos), *bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin, pos)]

    want = [step(t) for t in state]
    held = [[x.clone() if torch.is_tensor(x) else [y.clone() for y in x] for x in state[i]] for i in range(2)]
    graphs, outs = [], []
    for t in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(t))
        graphs.append(g)
    for pick in ((0, 1), (2, 3), (1, 0)):
        for t, i in zip(held, pick):
            for dst, src in zip(t, state[i]):
                for a, b in zip(dst if isinstance(dst, list) else [dst], src if isinstance(src, list) else [src]):
                    a.copy_(b)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for o, i in zip(outs, pick):
            assert all(torch.equal(x, y) for x, y in zip(o, want[i])), pick


def test_autograd_takes_the_kernels(cuda_device):
    q, k, qw, kw, cos, sin, _, dy = make(2, 33, 4, 2, 64, 16, BF16, FP32, seed=4, packed=False)
    leaves = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    y = training.qk_norm_rope(*leaves, cos, sin, nope_dim=0)
    want = norm.kernel_fn(q, k, qw, kw, cos, sin, nope_dim=0)
    assert all(torch.equal(a, b) for a, b in zip(y, want))
    torch.autograd.backward(y, dy)
    for leaf, g in zip(leaves, bwd.kernel_fn(*dy, q, k, qw, kw, cos, sin, nope_dim=0)):
        assert torch.equal(leaf.grad, g)
    # one output used, frozen weights
    q2 = q.clone().requires_grad_()
    training.qk_norm_rope(q2, k, qw, kw, cos, sin)[0].backward(dy[0])
    zero = torch.zeros_like(dy[1])
    assert torch.equal(q2.grad, bwd.kernel_fn(dy[0], zero, q, k, qw, kw, cos, sin)[0])
