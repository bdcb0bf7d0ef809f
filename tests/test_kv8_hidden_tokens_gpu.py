"""What a query row does not see must not reach it, finite or not: marked blocks and NaN bytes of later drafted tokens, in
kv8_attention and its checker."""

import math

import numpy as np
import pytest
import torch

from kernel_opt_agent_b200 import kv8_append as append
from kernel_opt_agent_b200 import kv8_attention as attention
from kernel_opt_agent_b200 import references
from tests.test_kv8_gpu import E4M3, GARBAGE_PAGE, INT8, _filled_cache, _i32, _pages, _queries


# sequence lengths whose newest tokens cross a page's border (and, in part, a tile's), heads that share a pass and not
CROSSING = [([33, 18], 3, 4, 2, 128, 16), ([49, 18], 3, 4, 2, 128, 16), ([65, 70, 3], 4, 2, 2, 64, 64), ([193, 130], 2, 8, 1, 256, 16),
            ([40], 16, 6, 2, 128, 32), ([433], 16, 6, 2, 128, 16), ([33, 49], 3, 16, 2, 64, 16), ([130, 260], 4, 12, 2, 256, 128)]


def _wide(cache, room):
    table = torch.cat([cache[4], torch.full((cache[4].shape[0], room), GARBAGE_PAGE, dtype=torch.int32, device=cache[4].device)], 1)
    return cache[:4] + [table]


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 4096])
@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("lens,t,hq,hkv,d,page", CROSSING)
def test_a_marked_page_of_later_tokens(cuda_device, cache_dtype, bad, room, lens, t, hq, hkv, d, page):
    """Drafted tokens open a new page, and the first of them there has a key (value) that is not finite: rows before it keep
    their bits, rows from it on are NaN, other heads and sequences keep theirs."""
    dev = cuda_device
    start = [max(n - t, 0) for n in lens]
    table, n = _pages(np.random.default_rng(d + t), lens, page)
    cache = append.make_cache(n, hkv, page, d, cache_dtype, dev) + [torch.from_numpy(table).to(dev)]
    gen = torch.Generator().manual_seed(t + hq)
    first = max(start)
    old = [torch.randn(len(lens), first, hkv, d, generator=gen).to(torch.bfloat16).to(dev) for _ in range(2)]
    append.kernel_fn(*old, *cache, _i32(start, dev), _i32(start, dev))
    k, v = (torch.randn(len(lens), t, hkv, d, generator=gen).to(torch.bfloat16).to(dev) for _ in range(2))
    q = _queries(t, len(lens), t, hq, d, torch.bfloat16, dev)
    seq, new = _i32(lens, dev), _i32([n - s for n, s in zip(lens, start)], dev)
    group = hq // hkv
    saved = [c.clone() for c in cache[:4]]
    append.kernel_fn(k, v, *cache, seq, new)
    want, want_lse = attention.kernel_fn(q, *_wide(cache, room), seq, new, return_lse=True)
    assert bool(want.isfinite().all())
    opens = -(-start[0] // page) * page  # the first new page of sequence 0
    assert start[0] < opens < lens[0], "the drafted tokens do not cross a page"
    i = opens - start[0]
    for which, (kk, vv) in (("v", (k, v.clone())), ("k", (k.clone(), v))):
        (vv if which == "v" else kk)[0, i, hkv - 1, 7] = bad
        for c, s in zip(cache, saved):
            c.copy_(s)
        append.kernel_fn(kk, vv, *cache, seq, new)
        out, lse = attention.kernel_fn(q, *_wide(cache, room), seq, new, return_lse=True)
        attention.check_device_status(dev)
        hit = torch.zeros(out.shape[:3], dtype=torch.bool, device=dev)
        hit[0, i:, (hkv - 1) * group:] = True
        assert bool(out[hit].isnan().all()), which
        assert torch.equal(out[~hit], want[~hit]), which
        assert torch.equal(lse[~hit], want_lse[~hit]), which
        ref = references.kv8_attention_ref(q, *cache, seq, new)
        assert torch.equal(ref.isnan(), hit[..., None].expand_as(ref)), which


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 4096])
@pytest.mark.parametrize("lens,t,hq,hkv,d,page", CROSSING)
def test_nan_bytes_of_later_tokens(cuda_device, room, lens, t, hq, hkv, d, page):
    """A cache of the caller's own with NaN bytes among the newest tokens' values: rows that see one are NaN in its
    dimension alone, rows that do not keep their bits."""
    dev = cuda_device
    cache = _wide(_filled_cache(sum(lens) + d, lens, hkv, d, page, E4M3, dev), room)
    q = _queries(t, len(lens), t, hq, d, torch.bfloat16, dev)
    seq, new = _i32(lens, dev), _i32([min(t, n) for n in lens], dev)
    bytes_ = cache[1].view(torch.uint8)
    group = hq // hkv
    marks = []  # page, head, slot, dim, row from which it is seen
    for i, h, dim in ((1, 0, 0), (t - 1, hkv - 1, d - 1), (t // 2, hkv - 1, 37), (t - 1, 0, 21)):
        pos = lens[0] - t + i
        marks.append((int(cache[4][0, pos // page]), h, pos % page, dim, i))
        bytes_[marks[-1][:4]] = 0
    want, want_lse = attention.kernel_fn(q, *cache, seq, new, return_lse=True)
    assert bool(want.isfinite().all())
    hit = torch.zeros(want.shape, dtype=torch.bool, device=dev)
    for x, (pid, h, slot, dim, i) in enumerate(marks):
        bytes_[pid, h, slot, dim] = 0x7F if x % 2 == 0 else 0xFF
        hit[0, i:, h * group:(h + 1) * group, dim] = True
    out, lse = attention.kernel_fn(q, *cache, seq, new, return_lse=True)
    attention.check_device_status(dev)
    assert torch.equal(out.isnan(), hit)
    assert torch.equal(out[~hit], want[~hit]) and torch.equal(lse, want_lse)
    ref = references.kv8_attention_ref(q, *cache[:4], cache[4], seq, new)
    assert torch.equal(ref.isnan(), hit)


def test_attention_checker_masks_before_it_multiplies():
    """CPU: the second of two tokens has a NaN value; the first row does not see it."""
    k_cache, v_cache, k_scale, v_scale = append.make_cache(1, 1, 16, 64, E4M3, device="cpu")
    v_cache.view(torch.uint8)[0, 0, 1, 3] = 0x7F
    k_scale.fill_(1.0)
    v_scale.fill_(1.0)
    q = torch.ones(1, 2, 1, 64, dtype=torch.bfloat16)
    table, seq = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    out, lse = references.kv8_attention_ref(q, k_cache, v_cache, k_scale, v_scale, table, seq, return_lse=True)
    assert bool((out[0, 0] == 0).all()) and bool(out[0, 1, 0, 3].isnan()) and int(out.isnan().sum()) == 1
    torch.testing.assert_close(lse[0, :, 0], torch.tensor([0.0, math.log(2.0)]))
