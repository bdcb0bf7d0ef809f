"""kv8_attention plugin module -- decode attention over the paged 8-bit key/value cache that
``kv8_append`` fills: the single-token step that ``flash_attention_2`` (prefill) has none of, with the
module contract of the reference's plugins (``kernels/__init__.py:3-8``).  The reference's attention is
prefill only.

    kernel_fn(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, new_lens=None,
              sm_scale=None, *, out=None, return_lse=False) -> out  (or (out, lse))

q [B, T, Hq, D] bf16 or fp16, 1 <= T <= 16: the queries of each sequence's newest tokens (one in a decode
step, a few when drafted tokens are verified), already appended to the cache.  Row i < new_lens[b] stands at
position seq_lens[b] - new_lens[b] + i and sees the positions up to its own; query head h reads key/value
head h // (Hq // Hkv); default scale 1 / sqrt(D).  out [B, T, Hq, D] in q's type, on the values the cache stands for:
maxima, sums and accumulation in fp32; q (scaled by a power of two per row) and each softmax weight times its
value scale enter the products as fp16, where what is under 2^-39 of a row's largest such product is lost.
Rows that see nothing (padding behind new_lens[b], empty sequences) are zero, their lse -inf.  ``lse``
[B, T, Hq] fp32 is the logarithm of the row's sum of exponentials, for joining with attention over other
tokens.  q may be a slice of a packed tensor.  The cache's layout and the
sequence tensors: ``_kv8``.

Lengths that do not fit the call or the table make the sequence's rows NaN, a table entry outside the pool
the rows that see it; a later call or ``check_device_status`` reports them as ``TokmixDeviceError``.  A prompt
goes through ``flash_attention_2`` (bf16, its own tokens only) and its keys and values into the cache with
``kv8_append``; a chunk of more than 16 tokens behind a cached prefix has no attention here.

``kernel_fn`` runs ``tokmix_kv8_attention`` (``csrc/kv8_attention.cu``), no fallback."""

from __future__ import annotations

import functools
import math

import torch

from . import _kv8, _lib
from ._kv8 import make_cache  # noqa: F401
from .kv8_append import check_device_status  # noqa: F401

KERNEL_TYPE = "kv8_attention"
MAX_TOKENS = 16


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(tokens: int, hq: int, hkv: int, d: int, batch: int, max_pages: int, page: int, device: int) -> int:
    """The workspace of a call's sizes on a device."""
    with torch.cuda.device(device):
        return _lib.load().tokmix_kv8_attention_workspace_bytes_for(tokens, hq, hkv, d, batch, max_pages, page)


def _overlap(out: torch.Tensor, q: torch.Tensor) -> bool:
    """Whether out (contiguous) reaches into the memory between q's first and last element."""
    last = sum((n - 1) * s for n, s in zip(q.shape, q.stride()))
    return q.numel() > 0 and out.data_ptr() < q.data_ptr() + 2 * (last + 1) and q.data_ptr() < out.data_ptr() + 2 * out.numel()


def kernel_fn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
              v_scale: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
              new_lens: torch.Tensor | None = None, sm_scale: float | None = None, *,
              out: torch.Tensor | None = None, return_lse: bool = False):
    cache = _kv8.cache_args(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, new_lens)
    batch, tokens, hq, d = q.shape
    if tokens > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} new tokens per sequence (got {tokens}); prompts go through "
                         "flash_attention_2")
    if hq == 0 or hq % cache.heads_kv != 0:
        raise ValueError("query heads must be a multiple of key/value heads")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(d)
    dev = q.device
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.device != dev:
        raise ValueError("out must be a contiguous tensor shaped and typed like q")
    elif out.untyped_storage().data_ptr() == q.untyped_storage().data_ptr() and _overlap(out, q):
        raise ValueError("out must not share memory with q")
    lse = torch.empty((batch, tokens, hq), dtype=torch.float32, device=dev) if return_lse else None
    q, qs = _kv8.token_strides(q)
    status = _lib.host_status_ptr(dev, "kv8")
    need = _workspace_bytes(max(tokens, 1), hq, cache.heads_kv, d, batch, cache.max_pages, cache.page_size, dev.index)
    ws = _lib.empty((need,), torch.uint8, dev) if need else None  # per call: calls may overlap on other streams
    rc = _lib.call_on(dev, _lib.load().tokmix_kv8_attention, q.data_ptr(), *qs, out.data_ptr(),
                      lse.data_ptr() if return_lse else None, tokens, hq, _kv8.IO_DTYPES[q.dtype], sm_scale,
                      _kv8.byref(cache), ws.data_ptr() if need else None, need, status, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "kv8_attention")
    _lib.after_host_status_launch(dev, "kv8")
    return (out, lse) if return_lse else out


def get_inputs(batch: int = 64, tokens: int = 1, seq_len: int = 4096, head_num: int = 16, head_num_kv: int = 2,
               head_dim: int = 256, page_size: int = 64, cache_dtype: torch.dtype = torch.float8_e4m3fn,
               dtype: torch.dtype = torch.bfloat16, seed: int = 42, device: str = "cuda") -> dict:
    """N(0,1) queries and a cache of N(0,1) keys and values (rounded to the cache's type at one scale), its
    pages in a shuffled order, from a seeded CPU generator."""
    gen = torch.Generator().manual_seed(seed)
    per = -(-seq_len // page_size)
    q = torch.randn(batch, tokens, head_num, head_dim, generator=gen).to(dtype)
    table = torch.randperm(batch * per, generator=gen).to(torch.int32).view(batch, per)
    scale = 2.0 ** -6 if cache_dtype == torch.float8_e4m3fn else 2.0 ** -4
    out = {"q": q.to(device)}
    for name in ("k_cache", "v_cache"):
        x = torch.randn(batch * per, head_num_kv, page_size, head_dim, generator=gen) / scale
        out[name] = (x if cache_dtype == torch.float8_e4m3fn else x.round().clamp(-127, 127)).to(cache_dtype).to(device)
    for name in ("k_scale", "v_scale"):
        out[name] = torch.full((batch * per, head_num_kv), scale, device=device)
    out["block_table"] = table.to(device)
    out["seq_lens"] = torch.full((batch,), seq_len, dtype=torch.int32, device=device)
    return out


def get_flops(batch: int = 64, tokens: int = 1, seq_len: int = 4096, head_num: int = 16, head_dim: int = 256) -> int:
    pairs = tokens * seq_len - tokens * (tokens - 1) // 2
    return 4 * batch * head_num * pairs * head_dim


def get_bytes(batch: int = 64, tokens: int = 1, seq_len: int = 4096, head_num: int = 16, head_num_kv: int = 2,
              head_dim: int = 256, element_size: int = 2) -> int:
    """The cached keys and values read once, q read and out written."""
    return 2 * batch * seq_len * head_num_kv * head_dim + 2 * batch * tokens * head_num * head_dim * element_size
