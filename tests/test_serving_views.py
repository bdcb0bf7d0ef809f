"""Views that the 8-bit cache's calls take: rows of packed tensors, buffers shared with the output."""

import ctypes

import pytest
import torch

from kernel_opt_agent_b200 import _kv8, _lib
from kernel_opt_agent_b200 import kv8_append as append
from kernel_opt_agent_b200 import kv8_attention as attention


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------------------------ views
def _packed_slices(dev="cpu"):
    """One token (or head) of a packed tensor whose rows are no multiple of 8 long: the strides of dimensions of size 1
    are odd, though nothing is read along them."""
    flat = torch.arange(4 * 1 * 2 * 67, device=dev).to(torch.bfloat16)
    return [flat.view(4, 1, 2, 67)[:1, :, :1, :64], flat.view(8, 67)[1:2].as_strided((1, 1, 1, 64), (67, 67, 67, 1), 0),
            flat.view(8, 67)[:1].as_strided((1, 1, 2, 64), (131, 131, 64, 1), 0), flat[1:].view(-1)[:128].view(1, 1, 2, 64)]


def test_token_strides_of_single_rows():
    for x in _packed_slices():
        y, strides = _kv8.token_strides(x)
        assert torch.equal(x, y) and y.data_ptr() % 16 == 0
        assert all(s % 8 == 0 and s >= 0 for s in strides), (x.stride(), strides)
    both = torch.zeros(2, 3, 12, 64, dtype=torch.bfloat16)[:, :, 4:8]  # read in place
    assert _kv8.token_strides(both)[0] is both and _kv8.token_strides(both)[1] == both.stride()[:3]


@pytest.mark.gpu
def test_single_rows_of_packed_tensors(cuda_device):
    dev = cuda_device
    table, seq = _i32([[1, 0]], dev), _i32([1], dev)
    for x in _packed_slices(dev):
        hkv = x.shape[2]
        a, b = (append.make_cache(2, hkv, 16, 64, device=dev) for _ in range(2))
        append.kernel_fn(x, x, *a, table, seq)
        append.kernel_fn(x.flatten().clone().view(x.shape), x.flatten().clone().view(x.shape), *b, table, seq)
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b))
        got = attention.kernel_fn(x, *a, table, seq)
        assert torch.equal(got, attention.kernel_fn(x.flatten().clone().view(x.shape), *a, table, seq))
    append.check_device_status(dev)


# ------------------------------------------------------------------------------------ the output's memory
def test_overlap_of_output_and_queries():
    buf = torch.zeros(4 * 512, dtype=torch.bfloat16)
    q = buf[:512].view(1, 2, 4, 64)
    for at, want in ((0, True), (8, True), (504, True), (512, False), (1024, False)):
        assert attention._overlap(buf[at:at + 512].view(q.shape), q) == want
        assert attention._overlap(q, buf[at:at + 512].view(q.shape)) == want
    packed = torch.zeros(2, 2, 12, 64, dtype=torch.bfloat16)[:, :, 4:8]
    assert not attention._overlap(buf[:1024].view(2, 2, 4, 64), packed) and attention._overlap(packed[:1, :1], packed)


@pytest.mark.gpu
def test_queries_and_output_in_one_buffer(cuda_device):
    """A step's buffer that holds both: taken where they are apart, refused where they overlap."""
    dev, shape = cuda_device, (2, 1, 4, 64)
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, 9, 2, 64, generator=gen).to(torch.bfloat16).to(dev) for _ in range(2))
    cache, table, seq = append.make_cache(2, 2, 16, 64, device=dev), _i32([[1], [0]], dev), _i32([9, 9], dev)
    append.kernel_fn(k, v, *cache, table, seq)
    q = torch.randn(shape, generator=gen).to(torch.bfloat16).to(dev)
    want = attention.kernel_fn(q, *cache, table, seq)
    n = q.numel()
    buf = torch.full((3 * n,), 7.0, dtype=torch.bfloat16, device=dev)
    for a, b in ((0, n), (2 * n, n), (0, 2 * n)):
        buf.fill_(7.0)
        one, two = buf[a:a + n].view(shape), buf[b:b + n].view(shape)
        one.copy_(q)
        assert attention.kernel_fn(one, *cache, table, seq, out=two) is two
        assert torch.equal(two, want) and torch.equal(one, q) and int((buf == 7).sum()) >= n
    for b in (0, 64, n - 64):
        with pytest.raises(ValueError, match="share"):
            attention.kernel_fn(buf[:n].view(shape), *cache, table, seq, out=buf[b:b + n].view(shape))
    append.check_device_status(dev)


# ------------------------------------------------------------------------------------ one cache for two
@pytest.mark.parametrize("same", ["k", "k_scale"])
def test_append_refuses_one_cache_for_keys_and_values(same):
    """The kernel would write both to the same bytes at once (refused on the host: no GPU is touched)."""
    sizes = dict(k_page_stride=2048, k_head_stride=1024, v_page_stride=2048, v_head_stride=1024, block_table=4096, table_stride=4,
                 seq_lens=4096, new_lens=None, num_pages=8, page_size=16, heads_kv=2, head_dim=64, dtype=_lib.DTYPE_E4M3, batch=1,
                 max_pages=4)
    ptrs = dict(k=4096, v=8192, k_scale=12288, v_scale=16384)
    ptrs["v" if same == "k" else "v_scale"] = ptrs[same]
    cache = _lib.Kv8Cache(*ptrs.values(), *sizes.values())
    x = ctypes.c_void_p(4096)
    rc = _lib.load().tokmix_kv8_append(x, 128, 128, 64, x, 128, 128, 64, 1, 0, ctypes.byref(cache), None, None)
    assert rc == _lib.TOKMIX_ERR_INVALID_ARGUMENT and "each" in _lib.last_error()
    none = _lib.load().tokmix_kv8_append(x, 128, 128, 64, x, 128, 128, 64, 0, 0, ctypes.byref(cache), None, None)
    assert none == _lib.TOKMIX_OK
