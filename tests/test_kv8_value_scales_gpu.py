"""kv8_attention where value scales differ by far more than a byte's range: a block counts by its softmax weight times its
scale, and only in the rows that see it."""

import math

import numpy as np
import pytest
import torch

from kernel_opt_agent_b200 import kv8_attention as attention
from kernel_opt_agent_b200 import references
from tests.test_kv8_gpu import E4M3, GARBAGE_PAGE, HALF_STEP, INT8, _filled_cache, _i32, _queries

pytestmark = pytest.mark.gpu
QMAX = {E4M3: 448.0, INT8: 127.0}


def _wide(cache, room):
    table = torch.cat([cache[4], torch.full((cache[4].shape[0], room), GARBAGE_PAGE, dtype=torch.int32, device=cache[4].device)], 1)
    return cache[:4] + [table]


def _assert_near(got, q, cache, seq, new, sm_scale=None):
    """Holds an output to the 64-bit one.  Per element, with p the softmax weights, s the largest sum_i |q_i k_ij| * sm_scale of
    the row, A = sum_j p_j |v_j|, N the tokens, E the largest |log2| of a value scale:
      half a step of the output type times |o|;  half a step of fp16 (2^-11) times A for the weights (times scales) rounded to fp16;
      those under 2^-39 of the row's largest p_j vs_j lost, each at most qmax of them: N 2^-39 qmax max_j(p_j vs_j);
      scores of D products in fp32: 2 D 2^-23 s of A;  exponents s + log2 scale rounded some times: 4 2^-23 (s + 1 + E) of A;
      sums of N / 8 terms in fp32 and joins: (N 2^-26 + 2^-20) A;  half a step of the output type's subnormals."""
    k_cache, v_cache, k_scale, v_scale, table = cache
    ref = references.kv8_attention_ref(q, k_cache, v_cache, k_scale, v_scale, table, seq, new, sm_scale, dtype=torch.float64)
    d, page, group = q.shape[3], k_cache.shape[2], q.shape[2] // k_cache.shape[1]
    scale = d ** -0.5 if sm_scale is None else sm_scale
    far = float(v_scale[v_scale != 0].abs().double().log2().abs().max())
    for b, (end, n) in enumerate(zip(seq.tolist(), new.tolist())):
        k = references.kv8_values(k_cache, k_scale, table, b, end, torch.float64).repeat_interleave(group, 0)
        v = references.kv8_values(v_cache, v_scale, table, b, end, torch.float64).repeat_interleave(group, 0)
        vs = v_scale[table[b, :-(-end // page)].long()].double().t().repeat_interleave(page, 1)[:, :end].repeat_interleave(group, 0)
        for i in range(n):
            m = end - n + i + 1
            s = torch.einsum("hd,hld->hl", q[b, i].double(), k[:, :m]) * scale
            size = (torch.einsum("hd,hld->hl", q[b, i].double().abs(), k[:, :m].abs()) * scale).amax(-1)[:, None]
            p = torch.softmax(s, -1)
            a = torch.einsum("hl,hld->hd", p, v[:, :m].abs())
            rel = 2.0 ** -11 + 2 * d * 2.0 ** -23 * size + 4 * 2.0 ** -23 * (size + 1 + far) + m * 2.0 ** -26 + 2.0 ** -20
            lost = m * 2.0 ** -39 * QMAX[v_cache.dtype] * (p * vs[:, :m].abs()).amax(-1)[:, None]
            tol = HALF_STEP[q.dtype] * ref[b, i].abs() + rel * a + lost
            tol = tol + (2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134)
            err = (got[b, i].double() - ref[b, i]).abs()
            assert bool((err <= tol).all()), (b, i, float((err / tol).max()))


@pytest.mark.parametrize("room", [0, 4096])
@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
@pytest.mark.parametrize("d,page,n", [(64, 16, 50), (128, 16, 70), (128, 64, 700), (256, 32, 90), (64, 64, 3000)])
def test_a_huge_block_without_weight(cuda_device, cache_dtype, d, page, n, room):
    """All values are 1 but those of some blocks, near 2^40, whose keys score 100 less: the rest's mean, 1, stays."""
    dev = cuda_device
    cache = _wide(_filled_cache(d + n, [n], 1, d, page, cache_dtype, dev), room)
    far = cache[4][0, 1:-(-n // page) - 1:3].long()
    for c, s in ((0, 2), (1, 3)):
        cache[c].view(torch.uint8).fill_(1 if cache_dtype == INT8 else 0x38)  # the value 1
        cache[s].fill_(1.0)
    cache[0].view(torch.uint8)[far] = 0
    cache[3][far, 0] = 2.0 ** 40
    q = torch.zeros(1, 1, 8, d, dtype=torch.float16, device=dev)
    q[..., 0] = 100.0  # scores 100 and, in the block, 0
    one = _i32([1], dev)
    out, lse = attention.kernel_fn(q, *cache, _i32([n], dev), one, sm_scale=1.0, return_lse=True)
    attention.check_device_status(dev)
    # 1, and some e^-100 2^40 (under 2^-100 each)
    assert bool(((out.float() - 1).abs() <= 2.0 ** -10).all()), float(out.float().min())
    _assert_near(out, q, cache, _i32([n], dev), one, sm_scale=1.0)


@pytest.mark.parametrize("room", [0, 4096])
@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
@pytest.mark.parametrize("lens,t,hq,hkv,d,page", [
    ([49, 40], 3, 4, 2, 128, 16), ([33], 4, 2, 2, 64, 16), ([193, 130], 2, 8, 1, 256, 16), ([433], 16, 6, 2, 128, 16)])
def test_a_huge_block_of_later_tokens(cuda_device, cache_dtype, room, lens, t, hq, hkv, d, page):
    """The page that the later drafted tokens open has values 2^40, 2^80 or 2^100 times the others': rows before it keep
    their bits."""
    dev = cuda_device
    cache = _wide(_filled_cache(d + t, lens, hkv, d, page, cache_dtype, dev), room)
    q = _queries(t, len(lens), t, hq, d, torch.bfloat16, dev)
    seq, new = _i32(lens, dev), _i32([t] * len(lens), dev)
    want, want_lse = attention.kernel_fn(q, *cache, seq, new, return_lse=True)
    opens = -(-(lens[0] - t) // page)  # the first page of sequence 0 that is new
    i = opens * page - (lens[0] - t)
    assert 0 < i < t
    pid, kept = int(cache[4][0, opens]), cache[3].clone()
    for far in (40, 80, 100):
        cache[3].copy_(kept)
        cache[3][pid] *= 2.0 ** far
        out, lse = attention.kernel_fn(q, *cache, seq, new, return_lse=True)
        assert torch.equal(out[0, :i], want[0, :i]) and torch.equal(out[1:], want[1:]) and torch.equal(lse, want_lse)
        _assert_near(out, q, cache, seq, new)


@pytest.mark.parametrize("room", [0, 4096])
@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
@pytest.mark.parametrize("far", [20, 28, 38, 60])
@pytest.mark.parametrize("lens,t,hq,hkv,d,page", [
    ([900, 33], 1, 8, 2, 128, 16), ([2500], 1, 4, 1, 64, 16), ([700, 64], 2, 16, 2, 256, 16), ([1500], 4, 24, 2, 64, 32), ([400], 3, 10, 2, 128, 128)])
def test_scales_far_apart(cuda_device, cache_dtype, far, lens, t, hq, hkv, d, page, room):
    """Value scales from 2^-far to 2^far in random order."""
    dev = cuda_device
    cache = _wide(_filled_cache(far + d, lens, hkv, d, page, cache_dtype, dev), room)
    gen = torch.Generator().manual_seed(far)
    cache[3].copy_(torch.exp2(torch.randint(-far, far + 1, cache[3].shape, generator=gen).float()))
    q = _queries(far, len(lens), t, hq, d, torch.bfloat16, dev)
    seq, new = _i32(lens, dev), _i32([t] * len(lens), dev)
    out = attention.kernel_fn(q, *cache, seq, new)
    assert torch.equal(out, attention.kernel_fn(q, *cache, seq, new))
    _assert_near(out, q, cache, seq, new)


@pytest.mark.parametrize("room", [0, 4096])
@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
def test_a_long_sequence_keeps_its_small_blocks(cuda_device, cache_dtype, room):
    """65536 tokens of weights 1 and e^-0.3 in turn, all of value 1, and blocks of scale 2^36 without weight: their mean is 1
    (twelve sequences share the pages, so that every warp has many tiles)."""
    dev, d, page, n, b = cuda_device, 128, 64, 65536, 12
    cache = _wide(_filled_cache(1, [n], 1, d, page, cache_dtype, dev), room)
    far, one = cache[4][0, 3:n // page:5].long(), 1 if cache_dtype == INT8 else 0x38
    cache[4] = cache[4].repeat(b, 1)
    k, v = cache[0].view(torch.uint8), cache[1].view(torch.uint8)
    k.zero_()
    k[..., 0] = one
    k[:, :, ::2, 1] = one
    k[far] = 0
    v.fill_(one)
    cache[2].fill_(1.0)
    cache[3].fill_(1.0)
    cache[3][far, 0] = 2.0 ** 36
    q = torch.zeros(b, 1, 4, d, dtype=torch.float16, device=dev)
    q[..., 0], q[..., 1] = 90.0, -0.3
    out = attention.kernel_fn(q, *cache, _i32([n] * b, dev), sm_scale=1.0)
    # half a step of fp16 for the output and for the weights e^-0.3, fp32 sums of 8192 terms a warp (2^-11 more)
    assert bool(((out.float() - 1).abs() <= 2.0 ** -10 + 2.0 ** -11).all()), float(out.float().min())


@pytest.mark.parametrize("room", [0, 4096])
def test_scales_of_every_kind(cuda_device, room):
    """Zero, subnormal, large, not powers of two, negative: a value is its byte times its scale, whatever that is."""
    dev, page, d = cuda_device, 16, 128
    lens = [200, 200, 200, 200, 200]
    cache = _wide(_filled_cache(77, lens, 2, d, page, INT8, dev), room)
    q = _queries(77, 5, 1, 8, d, torch.bfloat16, dev)
    rng = np.random.default_rng(5)
    for b, kinds in enumerate(([0.0, 1.0], [0.0], [2.0 ** -140, 2.0 ** -127, 0.0], [2.0 ** 119, 1.0, 2.0 ** -30], [0.7, -1.3, 3e-5, 1.9])):
        for p in range(-(-lens[b] // page)):
            cache[3][int(cache[4][b, p])] = float(rng.choice(kinds))
    seq, new = _i32(lens, dev), _i32([1] * 5, dev)
    out = attention.kernel_fn(q, *cache, seq, new)
    assert bool((out[1] == 0).all())
    for b in (0, 2, 3, 4):
        s = slice(b, b + 1)
        _assert_near(out[s], q[s], cache[:4] + [cache[4][s]], seq[s], new[s])


@pytest.mark.parametrize("room", [0, 4096])
def test_scales_at_the_end_of_the_range(cuda_device, room):
    """Bytes -1, 0 and 1 at scales up to 1.5 * 2^127 beside ordinary ones."""
    dev, page, d, lens = cuda_device, 16, 64, [100, 300, 40]
    cache = _wide(_filled_cache(78, lens, 1, d, page, INT8, dev), room)
    cache[1].copy_(cache[1].sign())
    q = _queries(78, 3, 1, 4, d, torch.bfloat16, dev)
    rng = np.random.default_rng(6)
    for b, kinds in enumerate(([2.0 ** 126, 1.0], [1.5 * 2.0 ** 127, 2.0 ** -100, 2.0 ** 20], [2.0 ** 127])):
        for p in range(-(-lens[b] // page)):
            cache[3][int(cache[4][b, p])] = float(rng.choice(kinds))
    seq, new = _i32(lens, dev), _i32([1] * 3, dev)
    out = attention.kernel_fn(q, *cache, seq, new)
    assert bool(out.isfinite().all())
    _assert_near(out, q, cache, seq, new)
