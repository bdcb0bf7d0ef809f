"""The paged 8-bit key/value cache on a B200: kv8_append against its definition bit for bit, kv8_attention
against 64-bit softmax attention on the values the cache stands for, and both as a serving loop uses them."""

import math

import numpy as np
import pytest
import torch

from kernel_opt_agent_b200 import _kv8, _lib, add_rms_norm_quant, references
from kernel_opt_agent_b200 import flash_attention_2 as fa2
from kernel_opt_agent_b200 import kv8_append as append
from kernel_opt_agent_b200 import kv8_attention as attention
from kernel_opt_agent_b200 import qkv_part_rope as rope
from kernel_opt_agent_b200.kernel_configs import KERNEL_CONFIGS

pytestmark = pytest.mark.gpu
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
GARBAGE_PAGE = 0x7FFFFFFF  # a table entry nothing may read


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _pages(rng, lens, page, spare=3, garbage=GARBAGE_PAGE):
    """A shuffled block table for sequences of these lengths; entries behind the last page are garbage."""
    need = [-(-n // page) for n in lens]
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(lens), max(need + [1]) + 2), garbage, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def _bits_equal(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def _random_bytes(gen, shape, dtype):
    """Every finite e4m3 value (or int8 -127 .. 127), with equal weight."""
    if dtype == INT8:
        return torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8)
    b = torch.randint(0, 254, shape, generator=gen).to(torch.uint8)
    return torch.where(b >= 127, b + 1, b).to(torch.uint8).view(E4M3)  # leaves out 0x7f and 0xff, the NaNs


def _filled_cache(seed, lens, hkv, d, page, dtype, dev, rng=None):
    """A cache with random bytes, scales that differ by page and head, and bytes behind each sequence's end (and in
    pages of nobody) that must not matter: e4m3 NaN, int8 -128."""
    rng = rng or np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    table, n = _pages(rng, lens, page)
    caches, scales = [], []
    for lo, hi in ((-9, -5), (-12, 4)):
        c = torch.full((n, hkv, page, d), -128 if dtype == INT8 else 0x7F, dtype=torch.int8)
        c = c if dtype == INT8 else c.view(torch.uint8).view(E4M3)
        for b, length in enumerate(lens):
            for p in range(-(-length // page)):
                k = min(page, length - p * page)
                c[table[b, p], :, :k] = _random_bytes(gen, (hkv, k, d), dtype)
        caches.append(c.to(dev))
        scales.append(torch.exp2(torch.randint(lo, hi, (n, hkv), generator=gen).float()).to(dev))
    return caches + scales + [torch.from_numpy(table).to(dev)]


def _queries(seed, b, t, hq, d, dtype, dev):
    gen = torch.Generator().manual_seed(seed + 7)
    return torch.randn(b, t, hq, d, generator=gen).to(dtype).to(dev)


def _assert_attention(got, lse, q, cache, seq, new=None, sm_scale=None):
    """Holds an output to the 64-bit one.  Per element, with A = sum_j p_j |v_j| (p the softmax weights), N the
    tokens, and S the largest sum_i |q_i k_ij| * sm_scale of the row:
      half a step of the output type times |o|;  half a step of fp16 (2^-11) times A for weights rounded to fp16,
      and weights under 2^-38 of the largest lost: N 2^-38 max |v|;
      a score of D products, each sum off by a step of fp32 (2^-23): a relative D 2^-23 S of every weight, in
      numerator and denominator (times 2), with the exponential's argument rounded: 4 2^-23 (S + 1) more;
      sums of N / 8 terms in fp32: N 2^-26 A;  some roundings of the joins: 2^-20 A.
    The logarithm of the sum: the score's error, N 2^-26, and a step of fp32 of its own size."""
    k_cache, v_cache, k_scale, v_scale, table = cache
    ref, ref_lse = references.kv8_attention_ref(q, k_cache, v_cache, k_scale, v_scale, table, seq, new, sm_scale,
                                                dtype=torch.float64, return_lse=True)
    batch, tokens, hq, d = q.shape
    hkv = k_cache.shape[1]
    scale = d ** -0.5 if sm_scale is None else sm_scale
    ends = seq.tolist()
    news = new.tolist() if new is not None else [tokens] * batch
    assert got.shape == q.shape and got.dtype == q.dtype
    for b, (end, n) in enumerate(zip(ends, news)):
        assert bool((got[b, n:] == 0).all()), b
        if lse is not None:
            assert bool((lse[b, n:] == -math.inf).all()), b
        if n == 0:
            continue
        k = references.kv8_values(k_cache, k_scale, table, b, end, torch.float64).repeat_interleave(hq // hkv, 0)
        v = references.kv8_values(v_cache, v_scale, table, b, end, torch.float64).repeat_interleave(hq // hkv, 0)
        s = torch.einsum("thd,hld->htl", q[b, :n].double(), k) * scale
        size = torch.einsum("thd,hld->htl", q[b, :n].double().abs(), k.abs()) * scale
        hidden = torch.arange(end, device=q.device) > (end - n + torch.arange(n, device=q.device))[:, None]
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        a = torch.einsum("htl,hld->thd", p, v.abs())
        top = size.masked_fill(hidden, 0).amax(-1).t()[..., None]                       # [t, h, 1]
        rel = 2.0 ** -11 + 2 * d * 2.0 ** -23 * top + 4 * 2.0 ** -23 * (top + 1) + end * 2.0 ** -26 + 2.0 ** -20
        big = v.abs().amax(1)[None]                                                     # [1, h, d]
        tol = HALF_STEP[q.dtype] * ref[b, :n].abs() + rel * a + end * 2.0 ** -38 * big
        if q.dtype == torch.float16:
            tol = tol + 2.0 ** -25  # half a step of fp16's subnormals
        err = (got[b, :n].double() - ref[b, :n]).abs()
        assert bool((err <= tol).all()), (b, float((err / tol).max()))
        if lse is not None:
            tol = d * 2.0 ** -23 * top[..., 0] + 4 * 2.0 ** -23 * (top[..., 0] + 1) + end * 2.0 ** -26 + \
                2.0 ** -22 * ref_lse[b, :n].abs() + 2.0 ** -20
            err = (lse[b, :n].double() - ref_lse[b, :n]).abs()
            assert bool((err <= tol).all()), (b, float((err / tol).max()))


# ------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
@pytest.mark.parametrize("lens,t,hkv,d,page", [
    ([0], 1, 1, 64, 16), ([15, 16, 17], 1, 2, 64, 16), ([0, 5, 63, 64], 1, 3, 256, 64), ([127, 128], 3, 2, 128, 128),
    ([0, 1, 30], 5, 1, 64, 32), ([0, 7, 64], 40, 2, 128, 64), ([3, 0, 100], 333, 2, 64, 16), ([100], 300, 1, 256, 128),
    ([1], 129, 2, 128, 128)])
def test_append_matches_definition(cuda_device, io, cache_dtype, lens, t, hkv, d, page):
    """Prefixes of several lengths, then chunks of t tokens (ragged where there is room): bytes and scales equal
    the definition's, everything else in the pool stays."""
    rng = np.random.default_rng(sum(lens) + t)
    gen = torch.Generator().manual_seed(t + d)
    ends = [n + t for n in lens]
    table, n = _pages(rng, ends, page)
    table = torch.from_numpy(table).to(cuda_device)
    cache = append.make_cache(n, hkv, page, d, cache_dtype, cuda_device)
    for c in cache[:2]:
        c.view(torch.uint8).fill_(0x7F)
    for s in cache[2:]:
        s.fill_(3.0)
    prefix = max(lens)
    if prefix:
        k, v = (torch.randn(len(lens), prefix, hkv, d, generator=gen).to(io).to(cuda_device) for _ in range(2))
        seq = _i32(lens, cuda_device)
        want = references.kv8_append_ref(k, v, *cache, table, seq, seq)
        append.kernel_fn(k, v, *cache, table, seq, seq)
        append.check_device_status(cuda_device)
        assert all(_bits_equal(a, b) for a, b in zip(cache, want))
    new = [t] + [int(rng.integers(0, t + 1)) for _ in lens[1:]]
    k, v = (torch.randn(len(lens), t, hkv, d, generator=gen) * f for f in (5.0, 0.3))  # keys raise the scales
    k, v = k.to(io).to(cuda_device), v.to(io).to(cuda_device)
    seq, newt = _i32([a + b for a, b in zip(lens, new)], cuda_device), _i32(new, cuda_device)
    want = references.kv8_append_ref(k, v, *cache, table, seq, newt)
    for again in range(2):  # the second time changes nothing
        got = append.kernel_fn(k, v, *cache, table, seq, newt)
        append.check_device_status(cuda_device)
        assert all(a is b for a, b in zip(got, cache))
        assert all(_bits_equal(a, b) for a, b in zip(cache, want)), again


@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
def test_append_token_by_token_is_near_one_append(cuda_device, cache_dtype):
    """130 tokens one at a time with growing magnitudes.  The scales are those of one append; an e4m3 value differs by
    at most one step of the subnormals, an int8 value by at most one step (1/2 + 1/4 + ... of the final one)."""
    dev, t, page = cuda_device, 130, 64
    gen = torch.Generator().manual_seed(3)
    k = torch.randn(2, t, 2, 128, generator=gen) * torch.exp2(torch.arange(t) / 16.0)[None, :, None, None]
    k = k.to(torch.bfloat16).to(dev)
    table = _i32([[3, 1, 0], [5, 2, 4]], dev)
    one, many = (append.make_cache(6, 2, page, 128, cache_dtype, dev) for _ in range(2))
    append.kernel_fn(k, -k, *one, table, _i32([t, t], dev))
    for i in range(t):
        append.kernel_fn(k[:, i:i + 1], -k[:, i:i + 1], *many, table, _i32([i + 1] * 2, dev))
    append.check_device_status(dev)
    assert torch.equal(one[2], many[2]) and torch.equal(one[3], many[3])
    for a, b in zip(one[:2], many[:2]):
        step = 1.0 if cache_dtype == INT8 else 2.0 ** -9
        assert float((a.float() - b.float()).abs().max()) <= step
        assert _bits_equal(a[:, :, -1], b[:, :, -1]) or cache_dtype == INT8


def test_append_values_that_are_not_finite_mark_their_block(cuda_device):
    dev = cuda_device
    table = _i32([[0, 1]], dev)
    for bad, io in ((math.nan, torch.bfloat16), (math.inf, torch.float16), (-math.inf, torch.bfloat16)):
        for cache_dtype in (E4M3, INT8):
            cache = append.make_cache(2, 2, 16, 64, cache_dtype, dev)
            k = torch.ones(1, 20, 2, 64, dtype=io, device=dev)
            v = k.clone()
            k[0, 3, 1, 9] = bad
            append.kernel_fn(k, v, *cache, table, _i32([20], dev))
            assert cache[2].isnan().tolist() == [[False, True], [False, False]] and not bool(cache[3].isnan().any())
            append.kernel_fn(v[:, :1], v[:, :1], *cache, table, _i32([21], dev))
            assert cache[2].isnan().tolist() == [[False, True], [False, False]]
            append.kernel_fn(v[:, :1], v[:, :1], *cache, table, _i32([1], dev))  # the page starts afresh
            assert not bool(cache[2].isnan().any())
    append.check_device_status(dev)


def test_append_reads_slices_and_writes_strided_caches(cuda_device):
    """New tokens as slices of a packed QKV tensor, keys and values in one pool: the same bytes as from copies."""
    dev, t, hkv, d, page = cuda_device, 21, 2, 64, 16
    gen = torch.Generator().manual_seed(5)
    qkv = torch.randn(3, t, 8 + 2 * hkv, d, generator=gen).to(torch.bfloat16).to(dev)
    k, v = qkv[:, :, 8:8 + hkv], qkv[:, :, 8 + hkv:]
    table, n = _pages(np.random.default_rng(0), [t] * 3, page)
    table = torch.from_numpy(table).to(dev)
    seq = _i32([t] * 3, dev)
    plain = append.make_cache(n, hkv, page, d, E4M3, dev)
    append.kernel_fn(k.contiguous(), v.contiguous(), *plain, table, seq)
    pool = torch.zeros(n, 2, hkv, page, d, dtype=torch.uint8, device=dev).view(E4M3)
    both = [pool[:, 0], pool[:, 1]] + [torch.zeros_like(s) for s in plain[2:]]
    append.kernel_fn(k, v, *both, table[:, :5], seq)
    odd = torch.empty(k.numel() + 1, dtype=k.dtype, device=dev)[1:].view(k.shape)
    odd.copy_(k)
    third = append.make_cache(n, hkv, page, d, E4M3, dev)
    append.kernel_fn(odd, v.expand(3, t, hkv, d), *third, table, seq)
    append.check_device_status(dev)
    for other in (both, third):
        assert all(_bits_equal(a.contiguous(), b.contiguous()) for a, b in zip(plain, other))


def test_append_nothing(cuda_device):
    cache = append.make_cache(2, 1, 16, 64, E4M3, cuda_device)
    before = [c.clone() for c in cache]
    k = torch.ones(1, 4, 1, 64, dtype=torch.bfloat16, device=cuda_device)
    table = _i32([[0, 1]], cuda_device)
    append.kernel_fn(k, k, *cache, table, _i32([9], cuda_device), _i32([0], cuda_device))
    append.kernel_fn(k[:, :0], k[:, :0], *cache, table, _i32([9], cuda_device))
    append.kernel_fn(k[:0], k[:0], *cache, table[:0], _i32([], cuda_device))
    append.check_device_status(cuda_device)
    assert all(_bits_equal(a, b) for a, b in zip(cache, before))


# ------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
@pytest.mark.parametrize("lens,t,hq,hkv,d,page,io", [
    ([1], 1, 1, 1, 64, 16, torch.bfloat16),
    ([1, 0, 2], 1, 4, 4, 128, 16, torch.float16),
    ([15, 16, 17, 33], 1, 4, 2, 64, 16, torch.bfloat16),
    ([63, 64, 65], 1, 16, 2, 256, 64, torch.bfloat16),
    ([129], 1, 16, 2, 256, 16, torch.bfloat16),
    ([127, 128, 129, 700], 1, 8, 1, 128, 32, torch.float16),
    ([1031, 5], 1, 5, 1, 64, 128, torch.bfloat16),
    ([300, 1], 1, 14, 2, 128, 64, torch.bfloat16),
    ([2000, 0, 31], 1, 12, 1, 256, 32, torch.float16),
    ([200], 1, 16, 1, 64, 64, torch.bfloat16),
    ([130, 90], 1, 40, 2, 128, 16, torch.bfloat16),
    ([5, 40, 77], 4, 8, 8, 64, 32, torch.float16),
    ([3, 200], 3, 16, 2, 256, 64, torch.bfloat16),
    ([16, 333], 16, 10, 2, 128, 16, torch.bfloat16),
    ([48], 16, 24, 1, 256, 128, torch.float16),
    ([5000, 4097], 1, 16, 2, 256, 64, torch.bfloat16),
    ([9000], 2, 8, 2, 128, 64, torch.bfloat16)])
def test_attention_matches_definition(cuda_device, cache_dtype, lens, t, hq, hkv, d, page, io):
    seed = sum(lens) + hq + d
    cache = _filled_cache(seed, lens, hkv, d, page, cache_dtype, cuda_device)
    q = _queries(seed, len(lens), t, hq, d, io, cuda_device)
    seq = _i32(lens, cuda_device)
    new = _i32([min(t, n) for n in lens], cuda_device)
    out, lse = attention.kernel_fn(q, *cache, seq, new, return_lse=True)
    attention.check_device_status(cuda_device)
    _assert_attention(out, lse, q, cache, seq, new)
    assert torch.equal(out, attention.kernel_fn(q, *cache, seq, new))      # the same bits again
    if min(lens) >= t:
        assert torch.equal(out, attention.kernel_fn(q, *cache, seq))
    # a table with room for much longer sequences takes the path that cuts sequences up
    wide = torch.cat([cache[4], torch.full((len(lens), 4096), GARBAGE_PAGE, dtype=torch.int32, device=cuda_device)], 1)
    out, lse = attention.kernel_fn(q, *cache[:4], wide, seq, new, return_lse=True)
    attention.check_device_status(cuda_device)
    _assert_attention(out, lse, q, cache, seq, new)
    assert torch.equal(out, attention.kernel_fn(q, *cache[:4], wide, seq, new))


def test_attention_many_ragged_sequences(cuda_device):
    """300 sequences of 0 to 400 tokens, padded rows of several lengths: every row, and the buffer around them."""
    rng = np.random.default_rng(11)
    lens = [int(x) for x in rng.integers(0, 400, 300)]
    lens[17] = lens[299] = 0
    cache = _filled_cache(2, lens, 2, 64, 32, E4M3, cuda_device, rng)
    q = _queries(2, 300, 3, 6, 64, torch.bfloat16, cuda_device)
    seq, new = _i32(lens, cuda_device), _i32([min(n, int(rng.integers(0, 4))) for n in lens], cuda_device)
    buf = torch.full((302, 3, 6, 64), 7.0, dtype=torch.bfloat16, device=cuda_device)
    out, lse = attention.kernel_fn(q, *cache, seq, new, out=buf[1:301], return_lse=True)
    attention.check_device_status(cuda_device)
    assert out.data_ptr() == buf[1:].data_ptr()
    _assert_attention(out, lse, q, cache, seq, new)
    # fewer sequences, so that each unit has a CTA of its own
    some = slice(0, 60)
    part, lse = attention.kernel_fn(q[some], *cache[:4], cache[4][some, :13], seq[some], new[some], return_lse=True)
    _assert_attention(part, lse, q[some], cache[:4] + [cache[4][some]], seq[some], new[some])
    assert bool((buf[0] == 7).all()) and bool((buf[301] == 7).all())


@pytest.mark.parametrize("cache_dtype,b,most,t,hq,hkv,d,page", [
    (E4M3, 40, 3000, 1, 8, 8, 64, 32), (INT8, 24, 2500, 1, 32, 8, 128, 64), (E4M3, 30, 2000, 3, 16, 4, 128, 16),
    (INT8, 9, 9000, 1, 16, 2, 256, 128), (E4M3, 5, 9000, 2, 24, 2, 256, 64), (E4M3, 2, 120000, 1, 8, 1, 64, 128)])
def test_attention_large_calls(cuda_device, cache_dtype, b, most, t, hq, hkv, d, page):
    """Calls that give every CTA many tiles and several units: every row, the same bits every time
    (also captured and replayed)."""
    rng = np.random.default_rng(b)
    lens = [most] + [int(x) for x in rng.integers(most // 2, most, b - 1)]
    lens[b // 2] = 0 if b > 3 else lens[b // 2]
    cache = _filled_cache(b, lens, hkv, d, page, cache_dtype, cuda_device, rng)
    q = _queries(b, b, t, hq, d, torch.bfloat16, cuda_device)
    seq, new = _i32(lens, cuda_device), _i32([min(t, n) for n in lens], cuda_device)
    out, lse = attention.kernel_fn(q, *cache, seq, new, return_lse=True)
    attention.check_device_status(cuda_device)
    _assert_attention(out, lse, q, cache, seq, new)
    for _ in range(5):
        assert torch.equal(out, attention.kernel_fn(q, *cache, seq, new))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = attention.kernel_fn(q, *cache, seq, new)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = attention.kernel_fn(q, *cache, seq, new)
    for _ in range(3):
        cap.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cap, out)
    assert torch.equal(other, out)




@pytest.mark.parametrize("sm_scale", [1e-6, 0.05, 30.0])
def test_attention_flat_and_sharp_softmax(cuda_device, sm_scale):
    lens = [700, 64]
    cache = _filled_cache(9, lens, 2, 128, 64, E4M3, cuda_device)
    q = _queries(9, 2, 1, 8, 128, torch.bfloat16, cuda_device)
    seq = _i32(lens, cuda_device)
    out, lse = attention.kernel_fn(q, *cache, seq, sm_scale=sm_scale, return_lse=True)
    _assert_attention(out, lse, q, cache, seq, sm_scale=sm_scale)


def test_attention_queries_of_every_size(cuda_device):
    """Zero queries average the values; very small and very large ones keep their scores."""
    lens = [200, 200, 200, 200]
    cache = _filled_cache(4, lens, 1, 64, 16, INT8, cuda_device)
    q = _queries(4, 4, 1, 8, 64, torch.bfloat16, cuda_device)
    q[0] = 0
    q[1] *= 1e-20
    q[2] *= 1e4
    q[3, 0, 0, :32] *= 1e-30
    seq = _i32(lens, cuda_device)
    _assert_attention(attention.kernel_fn(q, *cache, seq), None, q, cache, seq)


def test_attention_one_token_outweighs_a_long_flat_rest(cuda_device):
    """Weights far under the largest still add up: one score 14 above 60,000 equal ones."""
    n, d = 60001, 64
    cache = append.make_cache(-(-n // 128), 1, 128, d, INT8, cuda_device)
    cache[0][0, 0, 0] = 7
    cache[1].fill_(100)
    cache[1][0, 0, 0] = -100
    for s in cache[2:]:
        s.fill_(1.0)
    table = torch.arange(-(-n // 128), dtype=torch.int32, device=cuda_device)[None]
    q = torch.full((1, 1, 1, d), 0.25, dtype=torch.bfloat16, device=cuda_device)
    seq = _i32([n], cuda_device)
    out, lse = attention.kernel_fn(q, *cache, table, seq, return_lse=True)
    _assert_attention(out, lse, q, cache[:4] + [table], seq)


def test_attention_of_a_marked_block_is_nan(cuda_device):
    lens = [70, 70]
    cache = _filled_cache(6, lens, 2, 64, 16, E4M3, cuda_device)
    q = _queries(6, 2, 1, 4, 64, torch.bfloat16, cuda_device)
    seq = _i32(lens, cuda_device)
    want = attention.kernel_fn(q, *cache, seq)
    cache[2][int(cache[4][1, 2]), 0] = math.nan     # keys of sequence 1, head 0
    out = attention.kernel_fn(q, *cache, seq)
    assert bool(out[1, 0, :2].isnan().all())
    assert torch.equal(out[0], want[0]) and torch.equal(out[1, 0, 2:], want[1, 0, 2:])
    cache[3][int(cache[4][0, 1]), 1] = math.nan     # values of sequence 0, head 1
    out = attention.kernel_fn(q, *cache, seq)
    assert bool(out[0, 0, 2:].isnan().all()) and torch.equal(out[0, 0, :2], want[0, 0, :2])
    attention.check_device_status(cuda_device)


def test_attention_reads_slices_and_strided_caches(cuda_device):
    lens = [100, 37]
    cache = _filled_cache(8, lens, 2, 128, 32, E4M3, cuda_device)
    qkv = _queries(8, 2, 3, 12, 128, torch.bfloat16, cuda_device)
    q = qkv[:, :, :8]
    seq = _i32(lens, cuda_device)
    want = attention.kernel_fn(q.contiguous(), *cache, seq)
    n = cache[0].shape[0]
    pool = torch.empty(2, n, 2, 2, 32, 128, dtype=torch.uint8, device=cuda_device)
    pool[0, :, 0], pool[0, :, 1] = cache[0].view(torch.uint8), cache[1].view(torch.uint8)
    pool = pool.view(E4M3)
    heads_first = cache[1].view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(E4M3)
    assert torch.equal(attention.kernel_fn(q, pool[0, :, 0], pool[0, :, 1], *cache[2:], seq), want)
    assert torch.equal(attention.kernel_fn(q, cache[0], heads_first, *cache[2:], seq), want)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=cuda_device)[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(attention.kernel_fn(odd, *cache, seq), want)


def test_cache_beyond_two_gigabytes(cuda_device):
    """Pages whose byte offsets pass 2^31 and 2^32."""
    hkv, page, d = 8, 128, 256
    tile = hkv * page * d
    n = (1 << 32) // tile + 40
    free = torch.cuda.mem_get_info()[0]
    if free < 2.5 * n * tile:
        pytest.skip("not enough device memory")
    small = _filled_cache(12, [300, 170], hkv, d, page, E4M3, cuda_device)
    ids = torch.tensor([n - 1, (1 << 31) // tile, 0, (1 << 32) // tile + 1, n - 3, 5, (1 << 32) // tile, 9],
                       device=cuda_device)[:small[0].shape[0]]
    k, v = (torch.zeros(n, hkv, page, d, dtype=torch.uint8, device=cuda_device) for _ in range(2))
    ks, vs = (torch.ones(n, hkv, device=cuda_device) for _ in range(2))
    k[ids], v[ids], ks[ids], vs[ids] = small[0].view(torch.uint8), small[1].view(torch.uint8), small[2], small[3]
    valid = small[4] != GARBAGE_PAGE
    table = torch.where(valid, ids[torch.where(valid, small[4], 0).long()].int(), GARBAGE_PAGE)
    q = _queries(12, 2, 1, 16, d, torch.bfloat16, cuda_device)
    seq = _i32([300, 170], cuda_device)
    big = [k.view(E4M3), v.view(E4M3), ks, vs, table]
    assert torch.equal(attention.kernel_fn(q, *big, seq), attention.kernel_fn(q, *small, seq))
    x = torch.ones(2, 1, hkv, d, dtype=torch.bfloat16, device=cuda_device)
    append.kernel_fn(x, 2 * x, *big, _i32([301, 171], cuda_device))
    append.kernel_fn(x, 2 * x, *small, _i32([301, 171], cuda_device))
    seq = _i32([301, 171], cuda_device)
    assert torch.equal(attention.kernel_fn(q, *big, seq), attention.kernel_fn(q, *small, seq))
    append.check_device_status(cuda_device)


# ------------------------------------------------------------------------------------ errors
@pytest.mark.parametrize("room", [0, 4096])
def test_bad_pages_and_lengths_are_reported(cuda_device, room):
    """Table entries outside the pool and lengths that do not fit: nothing is read or written there, the other
    sequences are right, the error arrives at the next look and is gone after it.  (With and without room for long
    sequences in the table.)"""
    dev, lens, page = cuda_device, [40, 50, 60], 16
    cache = _filled_cache(13, lens, 2, 64, page, E4M3, dev)
    cache[4] = torch.cat([cache[4], torch.full((3, room), GARBAGE_PAGE, dtype=torch.int32, device=dev)], 1)
    q = _queries(13, 3, 1, 4, 64, torch.bfloat16, dev)
    seq = _i32(lens, dev)
    want = attention.kernel_fn(q, *cache, seq)
    attention.check_device_status(dev)
    for bad in (-1, cache[0].shape[0], GARBAGE_PAGE):
        table = cache[4].clone()
        table[1, 2] = bad
        out = attention.kernel_fn(q, *cache[:4], table, seq)
        with pytest.raises(_lib.TokmixDeviceError, match="argument"):
            attention.check_device_status(dev)
        attention.check_device_status(dev)
        assert bool(out[1].isnan().all()) and torch.equal(out[0], want[0]) and torch.equal(out[2], want[2])
        x = torch.ones(3, 1, 2, 64, dtype=torch.bfloat16, device=dev)
        mine = [c.clone() for c in cache[:4]]
        table[1, 3] = bad
        at = _i32([41, 49, 61], dev)
        ref = references.kv8_append_ref(x[::2], x[::2], *mine, table[::2], at[::2])
        append.kernel_fn(x, x, *mine, table, at)
        torch.cuda.synchronize()
        with pytest.raises(_lib.TokmixDeviceError):
            append.kernel_fn(x, x, *mine, cache[4], at)
        assert all(_bits_equal(a, b) for a, b in zip(mine, ref))
    capacity = cache[4].shape[1] * page
    for end, n in ((capacity + 1, 1), (-1, 1), (50, 2), (50, -1), (0, 1), (2 ** 31 - 1, 1)):
        s, new = _i32([40, end, 60], dev), _i32([1, n, 1], dev)
        out, lse = attention.kernel_fn(q, *cache, s, new, return_lse=True)
        with pytest.raises(_lib.TokmixDeviceError):
            attention.check_device_status(dev)
        assert bool(out[1].isnan().all()) and bool(lse[1].isnan().all())
        assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2])
        mine = [c.clone() for c in cache[:4]]
        x = torch.ones(3, 1, 2, 64, dtype=torch.bfloat16, device=dev)
        append.kernel_fn(x, x, *mine, cache[4], s, new)
        with pytest.raises(_lib.TokmixDeviceError):
            append.check_device_status(dev)
        ids = cache[4][1, :4].long()
        assert all(_bits_equal(a[ids], b[ids]) for a, b in zip(mine, cache[:4]))


def test_refusals(cuda_device):
    lens = [40, 50]
    cache = _filled_cache(14, lens, 2, 64, 16, E4M3, cuda_device)
    k_cache, v_cache, k_scale, v_scale, table = cache
    q, seq = _queries(14, 2, 1, 4, 64, torch.bfloat16, cuda_device), _i32(lens, cuda_device)
    k = q[:, :, :2].contiguous()
    for bad in [dict(q=q.float()), dict(q=q[0]), dict(q=q[..., :32]), dict(q=q[:, :, :3]), dict(q=q.repeat(1, 17, 1, 1)),
                dict(q=q.cpu()), dict(k_cache=k_cache.view(torch.uint8)), dict(v_cache=v_cache.view(INT8)),
                dict(v_cache=v_cache[:3]), dict(k_scale=k_scale.half()), dict(v_scale=v_scale.t()),
                dict(v_scale=v_scale[:, :1]), dict(block_table=table.long()), dict(block_table=table[:1]),
                dict(block_table=table.t().contiguous().t()), dict(seq_lens=seq.long()), dict(seq_lens=seq[:1]),
                dict(new_lens=seq[:1]), dict(new_lens=seq.cpu()), dict(sm_scale=-1.0), dict(sm_scale=math.nan),
                dict(out=q), dict(out=q.float()), dict(out=torch.empty_like(q)[:1]), dict(k_cache=k_cache.cpu())]:
        args = dict(q=q, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, block_table=table, seq_lens=seq)
        with pytest.raises(ValueError):
            attention.kernel_fn(**{**args, **bad})
    for bad in [dict(k=k.float()), dict(v=k.half()), dict(v=k[:, :, :1]), dict(k=q, v=q), dict(v=k.cpu()),
                dict(k=k[:1], v=k[:1]), dict(block_table=table[0])]:
        args = dict(k=k, v=k, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, block_table=table, seq_lens=seq)
        with pytest.raises(ValueError):
            append.kernel_fn(**{**args, **bad})
    attention.check_device_status(cuda_device)


def test_workspace_sizes(cuda_device):
    """A call needs no workspace with a short table; with room for long sequences it refuses less than it needs."""
    lib, lens = _lib.load(), [40, 50]
    cache = _filled_cache(15, lens, 2, 128, 16, E4M3, cuda_device)
    q, seq = _queries(15, 2, 1, 8, 128, torch.bfloat16, cuda_device), _i32(lens, cuda_device)
    want = attention.kernel_fn(q, *cache, seq)
    for room in (0, 4096):
        table = torch.cat([cache[4], torch.full((2, room), GARBAGE_PAGE, dtype=torch.int32, device=cuda_device)], 1)
        need = lib.tokmix_kv8_attention_workspace_bytes_for(1, 8, 2, 128, 2, table.shape[1], 16)
        most = lib.tokmix_kv8_attention_workspace_bytes(1, 8, 2, 128)
        assert need == (most if room else 0) and most > 0
        out = torch.zeros_like(q)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=cuda_device)
        desc = _kv8.cache_args(q, *cache[:4], table, seq, None)

        def call(ptr, size):
            return lib.tokmix_kv8_attention(q.data_ptr(), *q.stride()[:3], out.data_ptr(), None, 1, 8, 0, 128 ** -0.5,
                                            _kv8.byref(desc), ptr, size, None, _lib.stream_ptr(cuda_device))
        if room:
            assert call(None, need) == call(ws.data_ptr(), need - 1) == _lib.TOKMIX_ERR_INVALID_ARGUMENT
            assert call(ws.data_ptr(), need) == 0
        else:
            assert call(None, 0) == 0
            assert torch.equal(out, want)
        torch.cuda.synchronize()
        _assert_attention(out, None, q, cache, seq)


def test_refuses_more_sequences_or_tokens_than_int(cuda_device):
    cache = append.make_cache(2, 2, 16, 64, E4M3, cuda_device)
    one = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16, device=cuda_device)
    table, seq = _i32([[0, 1]], cuda_device), _i32([1], cuda_device)
    for k in (one.expand(2 ** 32 + 1, 1, 2, 64), one.expand(1, 2 ** 32 + 1, 2, 64)):  # one row of memory
        with pytest.raises(ValueError, match="2.31"):
            append.kernel_fn(k, k, *cache, table, seq)
        with pytest.raises(ValueError, match="2.31"):
            attention.kernel_fn(k, *cache, table, seq)


def test_empty_batches(cuda_device):
    cache = append.make_cache(2, 2, 16, 64, E4M3, cuda_device)
    q = torch.empty(0, 1, 4, 64, dtype=torch.bfloat16, device=cuda_device)
    none = _i32([], cuda_device)
    assert attention.kernel_fn(q, *cache, torch.empty(0, 3, dtype=torch.int32, device=cuda_device), none).shape == q.shape
    q = torch.ones(2, 1, 4, 64, dtype=torch.bfloat16, device=cuda_device)
    zero = _i32([0, 0], cuda_device)
    out, lse = attention.kernel_fn(q, *cache, torch.empty(2, 0, dtype=torch.int32, device=cuda_device), zero, zero,
                                   return_lse=True)
    attention.check_device_status(cuda_device)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    assert attention.kernel_fn(q[:, :0], *cache, _i32([[0], [1]], cuda_device), zero).shape == (2, 0, 4, 64)


@pytest.mark.parametrize("room", [0, 4096])
def test_query_rows_do_not_touch_each_other(cuda_device, room):
    """A NaN or infinite query spoils its own row, an empty sequence's rows are zero, all else keeps its bits."""
    lens = [100, 0, 37]
    cache = _filled_cache(40, lens, 2, 128, 32, E4M3, cuda_device)
    cache[4] = torch.cat([cache[4], torch.full((3, room), GARBAGE_PAGE, dtype=torch.int32, device=cuda_device)], 1)
    q = _queries(40, 3, 2, 8, 128, torch.bfloat16, cuda_device)
    seq, new = _i32(lens, cuda_device), _i32([2, 0, 2], cuda_device)
    want, want_lse = attention.kernel_fn(q, *cache, seq, new, return_lse=True)
    assert bool((want[1] == 0).all()) and bool((want_lse[1] == -math.inf).all())
    q[0, 1, 3, 5] = math.nan
    q[2, 0, 6, 0] = math.inf
    out, lse = attention.kernel_fn(q, *cache, seq, new, return_lse=True)
    attention.check_device_status(cuda_device)
    bad = torch.zeros(3, 2, 8, dtype=torch.bool, device=cuda_device)
    bad[0, 1, 3] = bad[2, 0, 6] = True
    assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], want[~bad]) and torch.equal(lse[~bad], want_lse[~bad])


def test_largest_batch(cuda_device):
    """8192 sequences that share pages: every one has what a call of few sequences gives; more are refused."""
    lens = [0, 70, 33, 128]
    cache = _filled_cache(41, lens, 1, 64, 64, INT8, cuda_device)
    q = _queries(41, 4, 1, 4, 64, torch.bfloat16, cuda_device)
    seq = _i32(lens, cuda_device)
    new = _i32([0, 1, 1, 1], cuda_device)
    want = attention.kernel_fn(q, *cache, seq, new)
    big = [q.repeat(2048, 1, 1, 1), *cache[:4], cache[4].repeat(2048, 1), seq.repeat(2048), new.repeat(2048)]
    out = attention.kernel_fn(*big)
    attention.check_device_status(cuda_device)
    # where a range border cuts a sequence: both outputs rounded (2 * 2^-8), both sets of weights rounded to fp16
    # (2 * 2^-11 of the largest value, 127 * 2^3)
    tol = 2.0 ** -7 * want.float().abs() + 2.0 ** -10 * 127 * 8
    assert bool(((out.view(2048, 4, 1, 4, 64).float() - want.float()).abs() <= tol).all())
    assert bool((out[::4] == 0).all())
    for i in (0, 5, 6, 8191):  # sequences whole inside a range are computed alike
        _assert_attention(out[i:i + 1], None, big[0][i:i + 1], cache[:4] + [big[5][i:i + 1]], big[6][i:i + 1], big[7][i:i + 1])
    more = [torch.cat([t, t[:1]]) for t in (big[0], big[5], big[6], big[7])]
    with pytest.raises(RuntimeError, match="8192"):
        attention.kernel_fn(more[0], *cache[:4], *more[1:])


@pytest.mark.parametrize("cache_dtype,b,t,hq,hkv,d,page,room", [
    (E4M3, 37, 1, 8, 1, 128, 32, 768), (E4M3, 38, 1, 8, 1, 128, 32, 1536), (INT8, 74, 1, 4, 1, 128, 64, 1536),
    (E4M3, 75, 1, 4, 1, 256, 16, 1536), (INT8, 148, 1, 4, 1, 64, 64, 6144), (E4M3, 149, 1, 4, 1, 64, 64, 2048),
    (E4M3, 149, 1, 4, 1, 64, 16, 2064), (INT8, 111, 1, 16, 4, 128, 128, 2048), (E4M3, 112, 1, 16, 4, 256, 32, 1024),
    (E4M3, 112, 1, 16, 4, 256, 32, 1056), (INT8, 90, 3, 20, 2, 128, 16, 2048), (E4M3, 300, 2, 16, 2, 64, 32, 2048),
    (E4M3, 9, 2, 16, 4, 64, 64, 2048), (E4M3, 10, 16, 3, 1, 256, 64, 512), (INT8, 150, 1, 4, 1, 128, 16, 1024),
    (E4M3, 150, 1, 4, 1, 128, 16, 1040), (E4M3, 333, 1, 8, 4, 128, 64, 2048), (INT8, 167, 1, 8, 2, 256, 16, 1024),
    (E4M3, 166, 1, 8, 2, 256, 16, 1024), (E4M3, 166, 1, 8, 2, 256, 16, 512)])
def test_attention_where_the_layout_changes(cuda_device, cache_dtype, b, t, hq, hkv, d, page, room):
    """Units (sequences times heads times row tiles) and room in the table on both sides of each border between the ways to lay
    the work out: one sequence fills its table, others are short or empty, one has nothing new."""
    rng = np.random.default_rng(b + d)
    lens = [int(x) for x in rng.integers(t, 150, b)]
    lens[b // 2], lens[1], lens[b - 1] = room, 0, t
    cache = _filled_cache(b, lens, hkv, d, page, cache_dtype, cuda_device, rng)
    table = torch.full((b, room // page), GARBAGE_PAGE, dtype=torch.int32, device=cuda_device)
    table[:] = cache[4][:, :room // page]
    cache[4] = table
    q = _queries(b, b, t, hq, d, torch.bfloat16, cuda_device)
    seq, new = _i32(lens, cuda_device), _i32([min(t, n) for n in lens[:2]] + [0] + [t] * (b - 3), cuda_device)
    out, lse = attention.kernel_fn(q, *cache, seq, new, return_lse=True)
    attention.check_device_status(cuda_device)
    _assert_attention(out, lse, q, cache, seq, new)
    assert torch.equal(out, attention.kernel_fn(q, *cache, seq, new))
    bad = seq.clone()
    bad[0] = room + 1
    out2, lse2 = attention.kernel_fn(q, *cache, bad, new, return_lse=True)
    with pytest.raises(_lib.TokmixDeviceError):
        attention.check_device_status(cuda_device)
    assert bool(out2[0].isnan().all()) and bool(lse2[0].isnan().all())
    _assert_attention(out2[1:], lse2[1:], q[1:], cache[:4] + [cache[4][1:]], seq[1:], new[1:])


@pytest.mark.parametrize("room", [0, 40])
def test_a_batch_of_thousands_of_units(cuda_device, room):
    """3000 sequences with 8 heads that share pages, as a CTA each or as ranges (room for 40 more pages): all have the bits or,
    where a range border cuts a sequence, nearly what a call of few sequences gives."""
    lens = [70, 33, 128]
    cache = _filled_cache(43, lens, 8, 64, 64, E4M3, cuda_device)
    q = _queries(43, 3, 1, 8, 64, torch.float16, cuda_device)
    seq = _i32(lens, cuda_device)
    want = attention.kernel_fn(q, *cache, seq)
    table = torch.cat([cache[4], torch.full((3, room), GARBAGE_PAGE, dtype=torch.int32, device=cuda_device)], 1)
    out = attention.kernel_fn(q.repeat(1000, 1, 1, 1), *cache[:4], table.repeat(1000, 1), seq.repeat(1000))
    attention.check_device_status(cuda_device)
    # both outputs rounded (2 * 2^-11 of it), both sets of weights rounded to fp16 (2 * 2^-11 of the largest value, 448 * 2^3)
    tol = 2.0 ** -10 * want.float().abs() + 2.0 ** -10 * 448 * 8
    assert bool(((out.view(1000, 3, 1, 8, 64).float() - want.float()).abs() <= tol).all())
    for i in (0, 1, 2, 1499, 2998, 2999):
        _assert_attention(out[i:i + 1], None, q[i % 3:i % 3 + 1], cache[:4] + [cache[4][i % 3:i % 3 + 1]], seq[i % 3:i % 3 + 1])


def test_largest_batch_in_ranges(cuda_device):
    """8192 sequences with room for long ones, so that the call is cut into ranges."""
    lens = [1, 70, 33, 128]
    cache = _filled_cache(42, lens, 1, 64, 64, INT8, cuda_device)
    q = _queries(42, 4, 1, 4, 64, torch.bfloat16, cuda_device)
    seq = _i32(lens, cuda_device)
    want = attention.kernel_fn(q, *cache, seq)
    table = torch.cat([cache[4], torch.full((4, 40), GARBAGE_PAGE, dtype=torch.int32, device=cuda_device)], 1)
    out = attention.kernel_fn(q.repeat(2048, 1, 1, 1), *cache[:4], table.repeat(2048, 1), seq.repeat(2048))
    attention.check_device_status(cuda_device)
    # both outputs rounded (2 * 2^-8), both sets of weights rounded to fp16 (2 * 2^-11 of the largest value, 127 * 2^3)
    tol = 2.0 ** -7 * want.float().abs() + 2.0 ** -10 * 127 * 8
    assert bool(((out.view(2048, 4, 1, 4, 64).float() - want.float()).abs() <= tol).all())
    for i in (0, 1, 2, 3, 4000, 8190, 8191):
        _assert_attention(out[i:i + 1], None, q[i % 4:i % 4 + 1], cache[:4] + [cache[4][i % 4:i % 4 + 1]], seq[i % 4:i % 4 + 1])


def test_append_extreme_magnitudes(cuda_device):
    """Scales at both ends: the largest bf16 values, and values under 2^-100 of a byte's reach, which become zeros."""
    table, seq = _i32([[0]], cuda_device), _i32([3], cuda_device)
    for dtype in (E4M3, INT8):
        for value in (3.3e38, 1e-36, 2.0 ** -95):
            k = torch.full((1, 3, 1, 64), value, dtype=torch.bfloat16, device=cuda_device)
            k[0, 1] = -k[0, 1]
            cache = append.make_cache(1, 1, 16, 64, dtype, cuda_device)
            want = references.kv8_append_ref(k, k, *cache, table, seq)
            append.kernel_fn(k, k, *cache, table, seq)
            assert all(_bits_equal(a, b) for a, b in zip(cache, want))
            assert bool(torch.isfinite(cache[2]).all()) and float(cache[2]) >= 2.0 ** -100
    append.check_device_status(cuda_device)


# ------------------------------------------------------------------------------------ streams, graphs
def test_two_streams_at_once(cuda_device):
    """Calls in flight on two streams have workspaces of their own."""
    cases = []
    for seed, lens in ((20, [9000, 3000]), (21, [5000, 8000])):
        cache = _filled_cache(seed, lens, 2, 128, 64, E4M3, cuda_device)
        cases.append((_queries(seed, 2, 1, 16, 128, torch.bfloat16, cuda_device), cache, _i32(lens, cuda_device)))
    want = [attention.kernel_fn(q, *c, s) for q, c, s in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (st, (q, c, s)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(st):
                got[i].append(attention.kernel_fn(q, *c, s))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


def test_captured_decode_steps(cuda_device):
    """Two graphs of append + attention, replayed side by side while lengths, tokens and queries change in place,
    against eager steps."""
    dev, page, hq, hkv, d, steps = cuda_device, 16, 8, 2, 128, 20
    append.check_device_status(dev)
    gen = torch.Generator().manual_seed(1)
    toks = torch.randn(2, steps, 3, 1, hq + 2 * hkv, d, generator=gen).to(torch.bfloat16).to(dev)
    sides = []
    for i, start in enumerate(([0, 15, 100], [64, 3, 0])):
        lens = [n + steps for n in start]
        cache = _filled_cache(30 + i, lens, hkv, d, page, E4M3, dev)
        cur = _i32(start, dev)
        qkv = torch.zeros(3, 1, hq + 2 * hkv, d, dtype=torch.bfloat16, device=dev)

        def step(cache=cache, cur=cur, qkv=qkv):
            cur.add_(1)
            append.kernel_fn(qkv[:, :, hq:hq + hkv], qkv[:, :, hq + hkv:], *cache, cur)
            return attention.kernel_fn(qkv[:, :, :hq], *cache, cur)

        start_state = [c.clone() for c in cache[:4]]
        want = []
        for t in range(steps):
            qkv.copy_(toks[i, t])
            want.append(step().clone())
        for c, s in zip(cache, start_state):
            c.copy_(s)
        cur.copy_(_i32(start, dev))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        cur.copy_(_i32(start, dev))
        sides.append((graph, out, qkv, want, torch.cuda.Stream(), [], (cache, cur)))  # the graph's tensors stay alive
    torch.cuda.synchronize()
    for t in range(steps):
        for i, (graph, out, qkv, want, st, got, _) in enumerate(sides):
            with torch.cuda.stream(st):
                qkv.copy_(toks[i, t])
                graph.replay()
                got.append(out.clone())
    torch.cuda.synchronize()
    append.check_device_status(dev)
    for _, _, _, want, _, got, _ in sides:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


# ------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("name", ["kv8_append", "kv8_attention"])
def test_config_sizes(cuda_device, name):
    cfg, mod = KERNEL_CONFIGS[name], {"kv8_append": append, "kv8_attention": attention}[name]
    for label, size in cfg["test_sizes"] + cfg["edge_sizes"]:
        for dtype in cfg["test_dtypes"]:
            inp = cfg["input_generator"](size, dtype, str(cuda_device))
            ref = cfg["reference_fn"](inp)
            got = mod.kernel_fn(**inp)
            pairs = zip(got, ref) if cfg.get("multi_output") else [(got, ref)]
            for g, r in pairs:
                assert g.shape == r.shape and g.dtype == r.dtype
                torch.testing.assert_close(g.float(), r.float(), **cfg["tolerances"][dtype], msg=label)
    append.check_device_status(cuda_device)


@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
def test_prompt_then_decode_with_the_packages_operators(cuda_device, cache_dtype):
    """One attention layer of a serving loop: residual norm to FP8 -> projection -> partial rotary embedding ->
    prompt attention (flash_attention_2) and its keys and values into the cache -> decode steps over the cache.
    Every decode step is held to 64-bit attention on what the cache stands for, and the cached values to the
    rotated keys and values they came from."""
    dev, b, prompt, steps, hq, hkv, d, page, n = cuda_device, 2, 100, 6, 8, 2, 128, 32, 256
    heads = hq + 2 * hkv
    gen = torch.Generator().manual_seed(17)
    weight = (torch.randn(heads * d, n, generator=gen) / 16).to(torch.bfloat16).to(dev)
    gamma = (1 + 0.1 * torch.randn(n, generator=gen)).to(torch.bfloat16).to(dev)
    hidden = torch.randn(b, prompt + steps, n, generator=gen).to(torch.bfloat16).to(dev)
    residual = torch.randn(b, prompt + steps, n, generator=gen).to(torch.bfloat16).to(dev)
    angle = torch.arange(prompt + steps, dtype=torch.float32)[:, None] * torch.exp2(-torch.arange(32) / 4.0)
    cos, sin = angle.cos().to(dev), angle.sin().to(dev)
    table, pages = _pages(np.random.default_rng(3), [prompt + steps] * b, page)
    table = torch.from_numpy(table).to(dev)
    cache = append.make_cache(pages, hkv, page, d, cache_dtype, dev)

    def project(lo, hi):
        x, r = hidden[:, lo:hi].contiguous(), residual[:, lo:hi].contiguous()
        y, scale, h = add_rms_norm_quant.kernel_fn(x, r, gamma)
        deq = y.float().view(-1, n // 128, 128) * scale.t()[..., None]
        qkv = (deq.view(-1, n).to(torch.bfloat16) @ weight.t()).view(b, hi - lo, heads, d)
        return rope.kernel_fn(qkv, cos[lo:hi].contiguous(), sin[lo:hi].contiguous(), q_heads=hq, kv_heads=hkv, nope_dim=64)

    packed = project(0, prompt)
    q, k, v = packed[:, :, :hq], packed[:, :, hq:hq + hkv], packed[:, :, hq + hkv:]
    prefill = fa2.kernel_fn(q.contiguous(), k.contiguous(), v.contiguous(), layout="bshd")
    append.kernel_fn(k, v, *cache, table, _i32([prompt] * b, dev))
    # the last prompt row over the cache is the prompt's own attention up to the 8-bit rounding of keys and values
    last = attention.kernel_fn(q[:, -1:], *cache, table, _i32([prompt] * b, dev), _i32([1] * b, dev))
    kk = [k]
    vv = [v]
    for t in range(prompt, prompt + steps):
        packed = project(t, t + 1)
        q1, k1, v1 = packed[:, :, :hq], packed[:, :, hq:hq + hkv], packed[:, :, hq + hkv:]
        seq = _i32([t + 1] * b, dev)
        append.kernel_fn(k1, v1, *cache, table, seq)
        out, lse = attention.kernel_fn(q1, *cache, table, seq, return_lse=True)
        _assert_attention(out, lse, q1, cache + [table], seq)
        kk.append(k1)
        vv.append(v1)
    append.check_device_status(dev)
    fa2.check_device_status(dev)
    for values, c, s in ((torch.cat(kk, 1), cache[0], cache[2]), (torch.cat(vv, 1), cache[1], cache[3])):
        for i in range(b):
            held = references.kv8_values(c, s, table, i, prompt + steps)
            true = values[i].float().transpose(0, 1)
            scale = s[table[i, :-(-(prompt + steps) // page)].long()].t().repeat_interleave(page, 1)[:, :prompt + steps, None]
            if cache_dtype == E4M3:  # half a step: 2^-4 of the value, or one subnormal step where rounded twice
                bound = (true.abs() * 2.0 ** -4).maximum(scale * 2.0 ** -9)
            else:                    # one step, however often rounded
                bound = scale.expand_as(true)
            assert bool(((held - true).abs() <= bound * 1.0001).all())
    # |o - o'| <= max |v - v'| + 2 max|v| * max |score change|; scores change by at most |q| |k - k'| / sqrt(d)
    for i in range(b):
        held_k = references.kv8_values(cache[0], cache[2], table, i, prompt)
        held_v = references.kv8_values(cache[1], cache[3], table, i, prompt)
        dk = (held_k - k[i].float().transpose(0, 1)).norm(dim=-1).amax()
        dv = (held_v - v[i].float().transpose(0, 1)).abs().amax()
        ds = q[i, -1].float().norm(dim=-1).amax() * dk / math.sqrt(d)
        vmax = v[i].float().abs().amax()
        bound = float(dv + vmax * (torch.exp(2 * ds) - 1)) + 2e-2 * (1 + float(vmax))
        assert float((last[i, 0].float() - prefill[i, -1].float()).abs().max()) <= bound
