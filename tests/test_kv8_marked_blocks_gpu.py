"""A value that is not finite marks its block in the 8-bit cache: a NaN scale over zero bytes, nothing else changed."""

import math

import numpy as np
import pytest
import torch

from kernel_opt_agent_b200 import kv8_append as append
from kernel_opt_agent_b200 import references
from tests.test_kv8_gpu import E4M3, INT8, _bits_equal, _i32, _pages


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
@pytest.mark.parametrize("io,bad", [(torch.bfloat16, math.nan), (torch.float16, math.inf), (torch.bfloat16, -math.inf)])
@pytest.mark.parametrize("t,hkv,d,page,old", [(1, 3, 64, 16, 0), (1, 2, 256, 64, 7), (20, 2, 64, 16, 5), (100, 1, 128, 64, 30), (333, 2, 256, 128, 3)])
def test_a_marked_block_gets_zero_bytes(cuda_device, cache_dtype, io, bad, t, hkv, d, page, old):
    """One value that is not finite: its block's scale is NaN, the new tokens' bytes there are zeros, and all else is what
    the append without that block is."""
    dev, gen = cuda_device, torch.Generator().manual_seed(t + d)
    table, n = _pages(np.random.default_rng(t), [old + t], page)
    table = torch.from_numpy(table).to(dev)
    k, v = (torch.randn(1, old + t, hkv, d, generator=gen).to(io).to(dev) for _ in range(2))
    cache = append.make_cache(n, hkv, page, d, cache_dtype, dev)
    if old:
        append.kernel_fn(k[:, :old], v[:, :old], *cache, table, _i32([old], dev))
    clean = [c.clone() for c in cache]
    k, v = k[:, old:].contiguous(), v[:, old:].contiguous()
    seq, new = _i32([old + t], dev), _i32([t], dev)
    append.kernel_fn(k, v, *clean, table, seq, new)
    at = (2 * t) // 3
    v[0, at, hkv - 1, d // 2] = bad
    want = references.kv8_append_ref(k, v, *cache, table, seq, new)
    append.kernel_fn(k, v, *cache, table, seq, new)
    append.check_device_status(dev)
    assert all(_bits_equal(a, b) for a, b in zip(cache, want))
    p = (old + at) // page
    pid = int(table[0, p])
    lo, hi = max(old - p * page, 0), min(old + t - p * page, page)
    assert math.isnan(float(cache[3][pid, hkv - 1])) and int(cache[3].isnan().sum()) == 1
    assert not bool(cache[1][pid, hkv - 1, lo:hi].view(torch.uint8).any())
    for a, b in zip(cache, clean):  # everything but that block
        a, b = a.clone(), b.clone()
        a.view(torch.uint8).view(n, hkv, -1)[pid, hkv - 1], b.view(torch.uint8).view(n, hkv, -1)[pid, hkv - 1] = 0, 0
        assert _bits_equal(a, b)


@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
def test_append_checker_zeroes_a_marked_block(cache_dtype):
    cache = append.make_cache(2, 1, 16, 64, cache_dtype, device="cpu")
    x = torch.ones(1, 20, 1, 64, dtype=torch.bfloat16)
    x[0, 18, 0, 5] = math.inf
    table, seq = torch.tensor([[1, 0]], dtype=torch.int32), torch.tensor([20], dtype=torch.int32)
    cache[0].view(torch.uint8).fill_(0x7F)
    k_cache, _, k_scale, _ = references.kv8_append_ref(x, x, *cache, table, seq)
    assert math.isnan(float(k_scale[0, 0])) and not bool(k_cache[0, 0, :4].view(torch.uint8).any())
    assert bool((k_cache[0, 0, 4:].view(torch.uint8) == 0x7F).all()) and bool((k_cache[1].float() != 0).all())
