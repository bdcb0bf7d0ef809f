"""kv8_append plugin module -- new keys and values enter a paged key/value cache held in 8 bits,
for ``kv8_attention`` to read; with the module contract of the reference's plugins
(``kernels/__init__.py:3-8``).  The reference has no cache (its attention is prefill only).

    kernel_fn(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, new_lens=None)
        -> [k_cache, v_cache, k_scale, v_scale]                      (updated in place)

k, v [B, T, Hkv, D] bf16 or fp16, any T (a decode step: 1; a prompt: its length).  Row i < new_lens[b]
becomes the token at position seq_lens[b] - new_lens[b] + i of sequence b; rows behind are padding.  k and v
may be slices of a packed tensor (``qkv_part_rope``'s output); they are read where they lie.
The cache's layout and the sequence tensors: ``_kv8``; ``make_cache`` allocates one.

Scales: per (page, head), for keys and values apart, the smallest power of two (at least 2^-100) with
max |x| <= qmax * scale over the page's tokens (qmax 448 for e4m3, 127 for int8).  When new tokens raise
a page's scale its older tokens are rounded again; a page whose first slot is written starts afresh,
so pages are reused without clearing.  A value that is not finite makes its block's scale NaN (the bytes
it brings are zeros): the whole block reads as NaN until the page starts afresh.

The caller keeps pages apart: a call appends to each page for one sequence, and at one place of its table (a
page shared by several sequences is full, or copied first), and k_cache and v_cache (k_scale and v_scale) are
not the same memory.  Lengths that do not fit the call or the table and table entries outside the pool write
nothing for that sequence (page) and are reported as ``TokmixDeviceError`` by a later call or by
``check_device_status``.

``kernel_fn`` runs ``tokmix_kv8_append`` (``csrc/kv8_append.cu``), no fallback."""

from __future__ import annotations

import torch

from . import _kv8, _lib
from ._kv8 import make_cache  # noqa: F401

KERNEL_TYPE = "kv8_append"


def kernel_fn(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
              v_scale: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
              new_lens: torch.Tensor | None = None) -> list[torch.Tensor]:
    cache = _kv8.cache_args(k, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, new_lens)
    if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError("k and v must have the same shape, type and device")
    if k.shape[2] != cache.heads_kv:
        raise ValueError("k and v must have the cache's heads")
    dev = k.device
    k, ks = _kv8.token_strides(k)
    v, vs = _kv8.token_strides(v)
    status = _lib.host_status_ptr(dev, "kv8")
    rc = _lib.call_on(dev, _lib.load().tokmix_kv8_append, k.data_ptr(), *ks, v.data_ptr(), *vs, k.shape[1],
                      _kv8.IO_DTYPES[k.dtype], _kv8.byref(cache), status, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "kv8_append")
    _lib.after_host_status_launch(dev, "kv8")
    return [k_cache, v_cache, k_scale, v_scale]


def check_device_status(device: torch.device | None = None) -> None:
    """Synchronise and raise if a kernel of the 8-bit cache met bad lengths or table entries on `device`."""
    idx = device.index if device is not None and device.index is not None else torch.cuda.current_device()
    torch.cuda.synchronize(idx)
    _lib.take_host_status(torch.device("cuda", idx), "kv8")


def get_inputs(batch: int = 64, tokens: int = 1, seq_len: int = 4096, head_num_kv: int = 2, head_dim: int = 256,
               page_size: int = 64, cache_dtype: torch.dtype = torch.float8_e4m3fn,
               dtype: torch.dtype = torch.bfloat16, seed: int = 42, device: str = "cuda") -> dict:
    """N(0,1) new tokens behind a cache of zeros (unit scales) of seq_len - tokens tokens per sequence, its
    pages in a shuffled order, from a seeded CPU generator."""
    gen = torch.Generator().manual_seed(seed)
    per = -(-seq_len // page_size)
    shape = (batch, tokens, head_num_kv, head_dim)
    k = torch.randn(shape, generator=gen).to(dtype)
    v = torch.randn(shape, generator=gen).to(dtype)
    table = torch.randperm(batch * per, generator=gen).to(torch.int32).view(batch, per)
    k_cache, v_cache, k_scale, v_scale = make_cache(batch * per, head_num_kv, page_size, head_dim, cache_dtype, device)
    k_scale.fill_(2.0 ** -8)
    v_scale.fill_(2.0 ** -8)
    return {"k": k.to(device), "v": v.to(device), "k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale,
            "v_scale": v_scale, "block_table": table.to(device),
            "seq_lens": torch.full((batch,), seq_len, dtype=torch.int32, device=device)}


def get_flops(batch: int = 64, tokens: int = 1, head_num_kv: int = 2, head_dim: int = 256) -> int:
    return 4 * batch * tokens * head_num_kv * head_dim


def get_bytes(batch: int = 64, tokens: int = 1, head_num_kv: int = 2, head_dim: int = 256,
              element_size: int = 2) -> int:
    """k and v read, their bytes written (the scales of the touched pages left out)."""
    return 2 * batch * tokens * head_num_kv * head_dim * (element_size + 1)
