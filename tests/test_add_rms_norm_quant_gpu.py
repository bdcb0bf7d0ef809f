"""add_rms_norm_quant on a B200 against its formula: the residual sum and the e4m3 bytes are exact, the
scales are held to a 64-bit evaluation."""

import pytest
import torch

from kernel_opt_agent_b200 import _lib, references
from kernel_opt_agent_b200 import add_rms_norm_quant as norm
from kernel_opt_agent_b200.kernel_configs import KERNEL_CONFIGS

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
# The scale is a * inv_rms / 448 with a exact.  The sum of n squares (all positive) passes through at most 64
# additions in a thread, 5 in a warp and 32 over warps, so it is off by at most 102 half steps of fp32 (2^-24);
# inv_rms carries half of that and five roundings of its own (mean, + eps, root, reciprocal, the square's),
# the scale two more: 58 * 2^-24, taken as 64.
SCALE_RTOL = 64 * 2.0 ** -24


def _inputs(dev, m, n, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed + m * 31 + n)
    return [t.to(dtype).to(dev) for t in (torch.randn(m, n, generator=gen), 4 * torch.randn(m, n, generator=gen),
                                          1 + 0.2 * torch.randn(n, generator=gen))]


def _check(x, r, w, group, got, eps=1e-6):
    y, scale, h = got
    ref_y, ref_scale, ref_h = references.add_rms_norm_quant_ref(x, r, w, eps, group)
    assert torch.equal(h, ref_h)
    assert y.shape == x.shape and y.dtype == torch.float8_e4m3fn
    assert torch.equal(y.view(torch.uint8), ref_y.view(torch.uint8))
    n = x.shape[-1]
    hd = ref_h.double().view(-1, n)
    inv = 1 / (hd.square().mean(-1, keepdim=True) + eps).sqrt()
    a = (hd * w.double()).view(hd.shape[0], -1, group or n).abs().amax(-1).clamp_min(2.0 ** -100)
    exact = a * inv / 448
    exact = exact.t() if group else exact.reshape(-1)
    assert scale.shape == exact.shape and scale.dtype == torch.float32
    torch.testing.assert_close(scale.double(), exact, rtol=SCALE_RTOL, atol=0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,group", [
    (1, 8, None), (5, 8, None), (3, 136, None), (1, 32, 32), (7, 96, 32), (1, 128, 128), (33, 128, 32),
    (9, 1024, 128), (4, 1032, None), (2, 2176, 128), (1, 4096, 128), (130, 4096, 32), (3, 4104, None),
    (5, 7168, 128), (2, 16384, 32), (2, 32768, None), (2, 32896, 128), (1, 65536, 128), (2, 65536, None)])
def test_matches_formula(cuda_device, dtype, m, n, group):
    x, r, w = _inputs(cuda_device, m, n, dtype)
    _check(x, r, w, group, norm.kernel_fn(x, r, w, group=group))


@pytest.mark.parametrize("name,size,dtype", [(label, size, dt) for c in [KERNEL_CONFIGS["add_rms_norm_quant"]]
                                             for label, size in c["test_sizes"] + c["edge_sizes"]
                                             for dt in c["test_dtypes"]], ids=lambda v: v if isinstance(v, str) else None)
def test_config_sizes(cuda_device, name, size, dtype):
    cfg = KERNEL_CONFIGS["add_rms_norm_quant"]
    inp = cfg["input_generator"](size, dtype, str(cuda_device))
    for g, r in zip(norm.kernel_fn(**inp), cfg["reference_fn"](inp)):
        assert g.shape == r.shape and g.dtype == r.dtype
        torch.testing.assert_close(g.float(), r.float(), **cfg["tolerances"][dtype])


@pytest.mark.parametrize("group", [None, 32, 128])
def test_without_residual_is_rms_norm(cuda_device, group):
    x, _, w = _inputs(cuda_device, 17, 768, torch.bfloat16)
    y, scale, h = norm.kernel_fn(x, None, w, group=group)
    assert h is x
    _check(x, None, w, group, (y, scale, h))
    g = group or 768
    got = y.float().view(17, -1, g) * (scale.t() if group else scale[:, None])[..., None]
    ref = references.rms_norm_ref(x.float(), w.float()).view(17, -1, g)
    # half a step of e4m3 relative (2^-4), half a step of its subnormals (2^-10) of the group's scale
    assert bool(((got - ref).abs() <= (ref.abs() * 2.0 ** -4 + ref.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -10) * 1.001).all())


def test_zero_tiny_and_large_groups(cuda_device):
    x, r, w = _inputs(cuda_device, 6, 256, torch.bfloat16)
    r.zero_()
    x[0] = 0                       # an empty row: bytes 0, scales finite
    x[1, :128] = 0                 # an empty group beside a full one
    x[2] = 1e-30
    x[3, 5] = 3e38                 # squares overflow: inv_rms = 0, every scale of the row is 0
    x[4, :] = -x[4, :].abs()
    y, scale, h = norm.kernel_fn(x, r, w)
    assert torch.equal(y.view(torch.uint8), references.add_rms_norm_quant_ref(x, r, w)[0].view(torch.uint8))
    assert bool((y[0].float() == 0).all()) and bool((y[1, :128].float() == 0).all())
    assert bool(torch.isfinite(scale).all()) and bool((scale[:, 3] == 0).all())
    assert bool((y[4].float() <= 0).all()) and float(y[4].float().min()) == -448


def test_values_that_are_not_finite_stay_in_their_row(cuda_device):
    for bad in (float("nan"), float("inf")):
        x, r, w = _inputs(cuda_device, 4, 256, torch.bfloat16)
        ok = norm.kernel_fn(x, r, w)
        x[2, 7] = bad
        y, scale, h = norm.kernel_fn(x, r, w)
        deq = y.float().view(4, 2, 128) * scale.t()[..., None]
        # NaN: the sum of squares makes every scale NaN; infinity: the group's scale (infinity times 0)
        assert bool(deq[2, 0].isnan().any())
        for i in (0, 1, 3):
            assert torch.equal(y[i].view(torch.uint8), ok[0][i].view(torch.uint8)) and torch.equal(scale[:, i], ok[1][:, i])


def test_inplace_shapes_strides_and_alignment(cuda_device):
    x, r, w = _inputs(cuda_device, 24, 256, torch.bfloat16)
    want = norm.kernel_fn(x, r, w)
    r2 = r.clone()
    y, scale, h = norm.kernel_fn(x, r2, w, inplace=True)
    assert h.data_ptr() == r2.data_ptr() and torch.equal(r2, want[2]) and torch.equal(scale, want[1])
    got = norm.kernel_fn(x.view(2, 3, 4, 256), r.view(2, 3, 4, 256), w)
    assert got[0].shape == (2, 3, 4, 256) and torch.equal(got[1], want[1]) and torch.equal(got[2].view(24, 256), want[2])
    wide = torch.empty(24, 512, dtype=x.dtype, device=cuda_device)
    wide[:, 100:356] = x
    odd = torch.empty(24 * 256 + 1, dtype=x.dtype, device=cuda_device)[1:].view(24, 256)
    odd.copy_(r)
    got = norm.kernel_fn(wide[:, 100:356], odd, w)
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[2], want[2])
    assert norm.kernel_fn(x[:0], r[:0], w)[1].shape == (2, 0)


def test_refusals(cuda_device):
    x, r, w = _inputs(cuda_device, 4, 256, torch.bfloat16)
    for bad in [lambda: norm.kernel_fn(x.float(), r.float(), w.float()), lambda: norm.kernel_fn(x, r.half(), w),
                lambda: norm.kernel_fn(x, r[:2], w), lambda: norm.kernel_fn(x, r, w[:128]),
                lambda: norm.kernel_fn(x, r, w, group=64), lambda: norm.kernel_fn(x[:, :160], r[:, :160], w[:160]),
                lambda: norm.kernel_fn(x, r.cpu(), w), lambda: norm.kernel_fn(x, r, w, eps=-1.0),
                lambda: norm.kernel_fn(x, None, w, inplace=True), lambda: norm.kernel_fn(x, r.t().contiguous().t(), w, inplace=True)]:
        with pytest.raises(ValueError):
            bad()


def test_refuses_more_rows_than_int_and_overlaps(cuda_device):
    w = torch.ones(8, dtype=torch.bfloat16, device=cuda_device)
    for rows in (2 ** 31 - 255, 2 ** 32 + 4):  # one row of memory
        with pytest.raises(ValueError, match="rows"):
            norm.kernel_fn(w.expand(rows, 8), None, w, group=None)
    buf = torch.randn(9, 256, device=cuda_device).to(torch.bfloat16)
    w = torch.ones(256, dtype=torch.bfloat16, device=cuda_device)
    for x, r in ((buf[1:], buf[:-1]), (buf[:-1], buf[1:])):
        with pytest.raises(ValueError, match="share no memory"):
            norm.kernel_fn(x, r, w, inplace=True)
    keep = buf.clone()
    got = norm.kernel_fn(buf[4:8], buf[:4], w, inplace=True)  # neighbours
    want = norm.kernel_fn(keep[4:8], keep[:4], w)
    assert torch.equal(buf[4:], keep[4:]) and torch.equal(got[2], want[2]) and torch.equal(got[1], want[1])
    same = keep[:4].clone()
    got = norm.kernel_fn(same, same, w, inplace=True)
    want = norm.kernel_fn(keep[:4], keep[:4], w)
    assert torch.equal(same, want[2]) and torch.equal(got[1], want[1])


def test_other_stream_and_graph(cuda_device):
    x, r, w = _inputs(cuda_device, 64, 4096, torch.bfloat16)
    want = norm.kernel_fn(x, r, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = norm.kernel_fn(x, r, w)
    side.synchronize()
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = norm.kernel_fn(x, r, w)
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    _check(x, r, w, 128, cap)


def test_launch_errors_are_reported(cuda_device):
    lib = _lib.load()
    assert lib.tokmix_add_rms_norm_quant(16, 16, 16, 16, 16, None, 4, 256, 128, 0, 1e-6, None) == 1
    assert "null" in _lib.last_error()
