"""The serving step's C entry points (tokmix_add_rms_norm_quant, tokmix_kv8_append, tokmix_kv8_attention)
reject bad arguments through their status codes without touching a GPU, and their checkers agree with
hand-made values (CPU only)."""

import ctypes
import math

import pytest
import torch

from kernel_opt_agent_b200 import _kv8, _lib, add_rms_norm_quant, kv8_append, kv8_attention, references

P = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(24)
INVALID, UNSUPPORTED, OK = _lib.TOKMIX_ERR_INVALID_ARGUMENT, _lib.TOKMIX_ERR_UNSUPPORTED, _lib.TOKMIX_OK


@pytest.mark.parametrize("changes,code", [
    (dict(rows=-1), INVALID), (dict(n=0), INVALID), (dict(n=100), UNSUPPORTED), (dict(n=192), UNSUPPORTED),
    (dict(n=65536 + 128), UNSUPPORTED), (dict(group=64), UNSUPPORTED), (dict(dtype=1), UNSUPPORTED),
    (dict(eps=-1.0), INVALID), (dict(eps=math.nan), INVALID), (dict(x=None), INVALID), (dict(weight=ODD), INVALID),
    (dict(residual_out=None), INVALID), (dict(y_scale=None), INVALID), (dict(rows=0), OK),
    (dict(group=32, n=48), UNSUPPORTED), (dict(group=0, n=12), UNSUPPORTED),
])
def test_norm_rejects_bad_arguments(changes, code):
    args = dict(x=P, residual=P, weight=P, residual_out=P, y=P, y_scale=P, rows=4, n=256, group=128, dtype=0,
                eps=1e-6, stream=None)
    args.update(changes)
    assert _lib.load().tokmix_add_rms_norm_quant(*args.values()) == code


@pytest.mark.parametrize("rows,code", [(2 ** 31 - 1, UNSUPPORTED), (2 ** 31 - 255, UNSUPPORTED)])
def test_norm_rejects_rows_its_indexes_do_not_hold(rows, code):
    assert _lib.load().tokmix_add_rms_norm_quant(P, P, P, P, P, P, rows, 256, 128, 0, 1e-6, None) == code


def _cache(**changes):
    c = dict(k=16, v=16, k_scale=16, v_scale=16, k_page_stride=16384, k_head_stride=8192, v_page_stride=16384,
             v_head_stride=8192, block_table=16, table_stride=4, seq_lens=16, new_lens=None, num_pages=8, page_size=64,
             heads_kv=2, head_dim=128, dtype=_lib.DTYPE_E4M3, batch=3, max_pages=4)
    c.update(changes)
    return _lib.Kv8Cache(*c.values())


BAD_CACHES = [
    (dict(k=None), INVALID), (dict(v_scale=None), INVALID), (dict(seq_lens=None), INVALID),
    (dict(block_table=None), INVALID), (dict(k=24), INVALID), (dict(k_page_stride=16392), INVALID),
    (dict(v_head_stride=4096), INVALID), (dict(num_pages=0), INVALID), (dict(heads_kv=0), INVALID),
    (dict(batch=-1), INVALID), (dict(table_stride=3), INVALID), (dict(page_size=48), UNSUPPORTED),
    (dict(page_size=256), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(dtype=0), UNSUPPORTED),
    (dict(max_pages=1 << 26, table_stride=1 << 26), UNSUPPORTED),
]


@pytest.mark.parametrize("cache,changes,code", [(c, {}, code) for c, code in BAD_CACHES] + [
    ({}, dict(tokens=-1), INVALID), ({}, dict(io=1), UNSUPPORTED), ({}, dict(k=None), INVALID), ({}, dict(v=ODD), INVALID),
    ({}, dict(kt=100), INVALID), ({}, dict(vh=-128), INVALID), ({}, dict(tokens=0), OK), (dict(batch=0), {}, OK),
])
def test_append_rejects_bad_arguments(cache, changes, code):
    args = dict(k=P, kb=256, kt=256, kh=128, v=P, vb=256, vt=256, vh=128, tokens=1, io=0)
    args.update(changes)
    c = _cache(**cache)
    assert _lib.load().tokmix_kv8_append(*args.values(), ctypes.byref(c), None, None) == code


@pytest.mark.parametrize("cache,changes,code", [(c, {}, code) for c, code in BAD_CACHES] + [
    ({}, dict(tokens=17), UNSUPPORTED), ({}, dict(tokens=-1), UNSUPPORTED), ({}, dict(hq=5), INVALID),
    ({}, dict(hq=0), INVALID), ({}, dict(io=1), UNSUPPORTED), ({}, dict(scale=0.0), INVALID),
    ({}, dict(scale=math.inf), INVALID), ({}, dict(q=None), INVALID), ({}, dict(out=ODD), INVALID),
    ({}, dict(qt=12), INVALID), ({}, dict(tokens=0), OK), (dict(batch=0), {}, OK),
])
def test_attention_rejects_bad_arguments(cache, changes, code):
    args = dict(q=P, qb=1024, qt=1024, qh=128, out=P, lse=None, tokens=1, hq=8, io=0, scale=0.1)
    args.update(changes)
    c = _cache(**cache)
    assert _lib.load().tokmix_kv8_attention(*args.values(), ctypes.byref(c), P, 1 << 40, None, None) == code


def test_null_cache_and_workspace_sizes():
    lib = _lib.load()
    assert lib.tokmix_kv8_append(P, 256, 256, 128, P, 256, 256, 128, 1, 0, None, None, None) == INVALID
    for bad in [(0, 8, 2, 128), (17, 8, 2, 128), (1, 7, 2, 128), (1, 8, 0, 128), (1, 8, 2, 96)]:
        assert lib.tokmix_kv8_attention_workspace_bytes(*bad) == -1


@pytest.mark.parametrize("bad", [(0, 8, 2, 128, 3, 4, 64), (1, 7, 2, 128, 3, 4, 64), (1, 8, 2, 96, 3, 4, 64), (1, 8, 2, 128, -1, 4, 64),
                                 (1, 8, 2, 128, 3, -1, 64), (1, 8, 2, 128, 3, 4, 0)])
def test_workspace_of_bad_sizes(bad):
    assert _lib.load().tokmix_kv8_attention_workspace_bytes_for(*bad) == -1
    assert _lib.load().tokmix_kv8_attention_workspace_bytes_for(1, 8, 2, 128, 0, 4, 64) == 0


def test_modules_refuse_cpu_tensors():
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        add_rms_norm_quant.kernel_fn(x, x, x[0])
    cache = kv8_append.make_cache(4, 2, 16, 64, device="cpu")
    k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    seq = torch.ones(1, dtype=torch.int32)
    table = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError):
        kv8_append.kernel_fn(k, k, *cache, table, seq)
    with pytest.raises(ValueError):
        kv8_attention.kernel_fn(k, *cache, table, seq)


def test_cache_strides_are_checked():
    """Views that share tiles, or tiles that are not contiguous, are refused; both caches in one tensor are not."""
    both = torch.zeros(5, 2, 3, 16, 64, dtype=torch.int8)
    assert _kv8._tile_strides("k", both[:, 0]) == (2 * 3 * 1024, 1024)
    assert _kv8._tile_strides("k", both[:1, 1, :1])[1] == 1024
    heads_first = torch.zeros(3, 5, 16, 64, dtype=torch.int8).transpose(0, 1)
    assert _kv8._tile_strides("k", heads_first) == (1024, 5 * 1024)
    tokens_first = torch.zeros(5, 16, 3, 64, dtype=torch.int8).transpose(1, 2)
    for bad in (tokens_first, both[:, 0, :1].expand(5, 3, 16, 64), both[:1, 0].expand(5, 3, 16, 64), both[:, 0, :, :, ::2],
                both.view(-1)[8:8 + 5 * 1024].view(5, 1, 16, 64)):
        with pytest.raises(ValueError):
            _kv8._tile_strides("k", bad)


def test_make_cache_refuses_sizes_without_a_kernel():
    for bad in [dict(page_size=48), dict(head_dim=96), dict(dtype=torch.uint8), dict(num_pages=0), dict(heads_kv=0)]:
        with pytest.raises(ValueError):
            kv8_append.make_cache(**{**dict(num_pages=4, heads_kv=2, device="cpu"), **bad})


@pytest.mark.parametrize("dtype,qmax", [(torch.float8_e4m3fn, 448.0), (torch.int8, 127.0)])
def test_append_checker_scales(dtype, qmax):
    """The scale is the smallest power of two that holds the page; it grows with new tokens, older bytes follow;
    a fresh page forgets its scale; a value that is not finite marks its block."""
    cache = kv8_append.make_cache(2, 1, 16, 64, dtype, device="cpu")
    table = torch.tensor([[1, 0]], dtype=torch.int32)

    def put(value, pos, cache):
        x = torch.full((1, 1, 1, 64), value, dtype=torch.bfloat16)
        return references.kv8_append_ref(x, -x, *cache, table, torch.tensor([pos + 1], dtype=torch.int32))

    cache = put(qmax * 2.0 ** -5, 0, cache) if dtype == torch.int8 else put(448.0 * 2.0 ** -5, 0, cache)
    assert float(cache[2][1, 0]) == 2.0 ** -5 and float(cache[0][1, 0, 0, 0].float()) == qmax
    big = 4.0 * qmax * 2.0 ** -5
    cache = put(big, 1, cache)
    assert float(cache[2][1, 0]) == 2.0 ** -3 and float(cache[0][1, 0, 1, 0].float()) == qmax
    held = float(cache[0][1, 0, 0, 0].float()) * 2.0 ** -3
    assert abs(held - qmax * 2.0 ** -5) <= 0.5 * 2.0 ** -3
    assert float(cache[3][1, 0]) == 2.0 ** -3 and float(cache[1][1, 0, 1, 5].float()) == -qmax
    cache = put(0.0, 0, cache)
    assert float(cache[2][1, 0]) == 2.0 ** -100
    cache = put(math.inf, 1, cache)
    assert math.isnan(float(cache[2][1, 0])) and math.isnan(float(cache[3][1, 0]))
    cache = put(1.0, 2, cache)
    assert math.isnan(float(cache[2][1, 0]))
    cache = put(1.0, 0, cache)
    assert float(cache[2][1, 0]) == (2.0 ** -8 if dtype == torch.float8_e4m3fn else 2.0 ** -6)


def test_attention_checker_on_a_hand_made_cache():
    """Two tokens with equal keys: the mean of their values; a second query row sees both, the first one only."""
    k_cache, v_cache, k_scale, v_scale = kv8_append.make_cache(1, 1, 16, 64, torch.int8, device="cpu")
    v_cache[0, 0, 0], v_cache[0, 0, 1] = 10, 30
    k_scale.fill_(1.0)
    v_scale.fill_(0.5)
    q = torch.ones(1, 2, 1, 64, dtype=torch.bfloat16)
    table, seq = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    out, lse = references.kv8_attention_ref(q, k_cache, v_cache, k_scale, v_scale, table, seq, return_lse=True)
    assert out[0, 0, 0, 0] == 5 and out[0, 1, 0, 0] == 10
    torch.testing.assert_close(lse[0, :, 0], torch.tensor([0.0, math.log(2.0)]))


@pytest.mark.parametrize("group", [None, 32, 128])
def test_norm_checker_dequantises_to_the_norm(group):
    gen = torch.Generator().manual_seed(1)
    x, r = (torch.randn(5, 256, generator=gen).to(torch.bfloat16) for _ in range(2))
    w = torch.randn(256, generator=gen).to(torch.bfloat16)
    y, scale, h = references.add_rms_norm_quant_ref(x, r, w, group=group)
    assert torch.equal(h, (x.float() + r.float()).to(torch.bfloat16))
    g = group or 256
    got = y.float().view(5, -1, g) * (scale.t() if group else scale[:, None])[..., None]
    ref = references.rms_norm_ref(h.float(), w.float()).view(5, -1, g)
    # e4m3: half a step (2^-4 relative), and half a step of its subnormals (2^-10) of the group's scale
    bound = ref.abs() * 2.0 ** -4 + ref.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -10 * 1.001
    assert bool(((got - ref).abs() <= bound * (1 + 1e-5)).all())
