"""What the plugin modules over the paged 8-bit key/value cache share: its layout, the checks of its
tensors, and the C description (``tokmix_kv8_cache``) they pass on.

A cache is four tensors: ``k_cache`` and ``v_cache`` [num_pages, Hkv, page, D] (float8_e4m3fn or int8)
and ``k_scale`` and ``v_scale`` [num_pages, Hkv] fp32; a cached value is byte * scale.  ``page`` is 16,
32, 64 or 128 tokens, D 64, 128 or 256.  The page and head dimensions may be strided (both caches in one
allocation, for instance); a [page, D] tile is contiguous.  A call names its sequences by ``block_table`` [B, max_pages]
int32 (a sequence's pages in order), ``seq_lens`` [B] int32 (tokens in the cache, this call's
included) and ``new_lens`` [B] int32 (how many of them are this call's; None: all T rows).
They stay on the device, so a call can be captured into a graph and replayed as they change."""

from __future__ import annotations

import ctypes

import torch

from . import _lib

CACHE_DTYPES = {torch.float8_e4m3fn: _lib.DTYPE_E4M3, torch.int8: _lib.DTYPE_INT8}
IO_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)


def make_cache(num_pages: int, heads_kv: int, page_size: int = 64, head_dim: int = 128,
               dtype: torch.dtype = torch.float8_e4m3fn, device="cuda"):
    """An empty cache: [k_cache, v_cache, k_scale, v_scale]."""
    if dtype not in CACHE_DTYPES or page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
        raise ValueError(f"a cache is {tuple(CACHE_DTYPES)}, page_size {PAGE_SIZES}, head_dim {HEAD_DIMS}")
    if num_pages < 1 or heads_kv < 1:
        raise ValueError("num_pages and heads_kv must be positive")
    kv = torch.zeros((2, num_pages, heads_kv, page_size, head_dim), dtype=torch.uint8, device=device).view(dtype)
    scale = torch.zeros((2, num_pages, heads_kv), dtype=torch.float32, device=device)
    return [kv[0], kv[1], scale[0], scale[1]]


def _tile_strides(name: str, t: torch.Tensor, shape=None) -> tuple[int, int]:
    """(page, head) strides of a cache; refuses tiles that are not contiguous, aligned or apart."""
    pages, heads, page, d = shape or t.shape
    sp, sh, ss, sd = t.stride()
    tile = page * d
    if sd == 1 and ss == d and sh == tile and sp == tile * heads and t.data_ptr() % 16 == 0:
        return sp, sh  # contiguous
    if pages == 1:
        sp = max(sp, tile * heads) // 16 * 16
    if heads == 1:
        sh = tile
    near, far = ((sh, heads), (sp, pages)) if sh <= sp else ((sp, pages), (sh, heads))
    if sd != 1 or ss != d or sp % 16 or sh % 16 or t.data_ptr() % 16 or near[0] < tile or (
            pages > 1 and heads > 1 and far[0] < near[0] * near[1]):
        raise ValueError(f"{name} must be [num_pages, Hkv, page, D] with contiguous, 16-byte aligned [page, D] tiles "
                         "that do not overlap")
    return sp, sh


def cache_args(x: torch.Tensor, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, new_lens) -> _lib.Kv8Cache:
    """Checks a cache and a call's sequences against x [B, T, heads, D] (the new keys or the queries)."""
    shape = k_cache.shape
    if x.ndim != 4 or len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("new tokens must be [B, T, heads, D], k_cache and v_cache [num_pages, Hkv, page, D]")
    num_pages, heads, page, d = shape
    batch, tokens = x.shape[:2]
    if batch >= 1 << 31 or tokens >= 1 << 31:
        raise ValueError("fewer than 2^31 sequences and new tokens per sequence")
    dtype = CACHE_DTYPES.get(k_cache.dtype)
    if dtype is None or v_cache.dtype != k_cache.dtype:
        raise ValueError("k_cache and v_cache must both be float8_e4m3fn or both int8")
    if page not in PAGE_SIZES or d not in HEAD_DIMS or num_pages == 0 or heads == 0:
        raise ValueError(f"page size must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}")
    if x.dtype not in IO_DTYPES or x.shape[3] != d:
        raise ValueError("new tokens must be bfloat16 or float16 with the cache's head_dim")
    dev = x.device
    if not x.is_cuda or k_cache.device != dev or v_cache.device != dev or k_scale.device != dev or (
            v_scale.device != dev or block_table.device != dev or seq_lens.device != dev) or (
            new_lens is not None and new_lens.device != dev):
        raise ValueError("all tensors must be CUDA tensors on one device")
    f32, i32, per_page = torch.float32, torch.int32, (num_pages, heads)
    if k_scale.dtype != f32 or v_scale.dtype != f32 or k_scale.shape != per_page or v_scale.shape != per_page or not (
            k_scale.is_contiguous() and v_scale.is_contiguous()):
        raise ValueError("k_scale and v_scale must be contiguous float32 [num_pages, Hkv]")
    if block_table.dtype != i32 or block_table.ndim != 2 or block_table.shape[0] != batch:
        raise ValueError("block_table must be int32 [B, max_pages]")
    max_pages = block_table.shape[1]
    table_stride, along = block_table.stride()
    if batch <= 1:
        table_stride = max_pages
    if table_stride < max_pages or (along != 1 and max_pages > 1):
        raise ValueError("the rows of block_table must be contiguous and must not overlap")
    if seq_lens.dtype != i32 or seq_lens.shape != (batch,) or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be contiguous int32 [B]")
    if new_lens is not None and (new_lens.dtype != i32 or new_lens.shape != (batch,) or not new_lens.is_contiguous()):
        raise ValueError("new_lens must be contiguous int32 [B]")
    kp, kh = _tile_strides("k_cache", k_cache, shape)
    vp, vh = _tile_strides("v_cache", v_cache, shape)
    return _lib.Kv8Cache(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), kp, kh, vp,
                         vh, block_table.data_ptr(), table_stride, seq_lens.data_ptr(),
                         new_lens.data_ptr() if new_lens is not None else None, num_pages, page, heads, d, dtype,
                         batch, max_pages)


def token_strides(x: torch.Tensor) -> tuple[torch.Tensor, tuple[int, int, int]]:
    """x [B, T, heads, D] and its (batch, token, head) strides if the kernels can read them in place
    (a slice of a packed QKV tensor, say), else a contiguous copy and the copy's."""
    sb, st, sh, sd = x.stride()
    if sd != 1 or (sb | st | sh) % 8 or x.data_ptr() % 16:
        # nothing is read along a dimension of size 1, whatever its stride
        sb, st, sh = (s if n > 1 else x.shape[3] for s, n in zip((sb, st, sh), x.shape))
        if sd != 1 or (sb | st | sh) % 8 or x.data_ptr() % 16:
            x = x.clone(memory_format=torch.contiguous_format)
            sb, st, sh, _ = x.stride()
    return x, (sb, st, sh)


def byref(c: _lib.Kv8Cache):
    return ctypes.byref(c)
