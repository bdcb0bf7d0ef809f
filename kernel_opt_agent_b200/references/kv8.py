"""Checkers of the paged 8-bit key/value cache: tokens appended one page at a time with power-of-two
scales (kv8_append) and softmax attention in fp32 on the values the cache stands for (kv8_attention)."""

from __future__ import annotations

import math

import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def _round(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return x.to(dtype) if dtype == torch.float8_e4m3fn else x.round().to(dtype)


def _scale_of(amax: float, qmax: float) -> float:
    """The smallest power of two, at least 2^-100, with amax <= qmax * scale; NaN if amax is not finite."""
    if not math.isfinite(amax):
        return math.nan
    e = max(-100, math.frexp(amax / qmax)[1] - 1 if amax else -100)  # 2^e <= amax / qmax < 2^(e + 1)
    return 2.0 ** e if amax <= qmax * 2.0 ** e else 2.0 ** (e + 1)


def _append_page(cache, scale, pid, h, lo, hi, x):
    """x [hi - lo, D] becomes slots lo .. hi - 1 of (page, head)."""
    s_old = float(scale[pid, h]) if lo > 0 else 0.0
    s = _scale_of(float(x.float().abs().amax()), QMAX[cache.dtype])
    s = math.nan if math.isnan(s) or math.isnan(s_old) else max(s, s_old)
    tile = cache[pid, h]
    if math.isnan(s):
        tile[lo:hi] = torch.zeros_like(x, dtype=torch.float32).to(cache.dtype)
    else:
        if s_old < s:
            tile[:lo] = _round(tile[:lo].float() * (s_old / s), cache.dtype)
        tile[lo:hi] = _round(x.float() / s, cache.dtype)
    scale[pid, h] = s


def kv8_append_ref(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, new_lens=None):
    """Updated copies of the cache and its scales.  (A block whose scale is NaN reads as NaN; its new bytes are zeros.)"""
    out = [t.clone() for t in (k_cache, v_cache, k_scale, v_scale)]
    page = k_cache.shape[2]
    ends = seq_lens.tolist()
    news = new_lens.tolist() if new_lens is not None else [k.shape[1]] * len(ends)
    table = block_table.tolist()
    for b, (end, n) in enumerate(zip(ends, news)):
        for p in range((end - n) // page, -(-end // page)):
            lo, hi = max(end - n - p * page, 0), min(end - p * page, page)
            if lo >= hi:
                continue
            i = p * page + lo - (end - n)
            for h in range(k_cache.shape[1]):
                _append_page(out[0], out[2], table[b][p], h, lo, hi, k[b, i:i + hi - lo, h])
                _append_page(out[1], out[3], table[b][p], h, lo, hi, v[b, i:i + hi - lo, h])
    return out


def kv8_values(cache, scale, block_table, b: int, length: int, dtype: torch.dtype = torch.float32):
    """The first `length` cached values of sequence b, [Hkv, length, D]."""
    page = cache.shape[2]
    ids = block_table[b, :-(-length // page)].long()
    x = cache.view(torch.uint8)[ids].view(cache.dtype).to(dtype) * scale[ids].to(dtype)[..., None, None]
    return x.transpose(0, 1).flatten(1, 2)[:, :length]


def kv8_attention_ref(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, new_lens=None, sm_scale=None,
                      dtype: torch.dtype = torch.float32, return_lse: bool = False):
    """softmax(q k^T sm_scale) v with the rows' causal limits, in `dtype`; out in q's type (or `dtype`, if wider
    than fp32)."""
    batch, tokens, hq, d = q.shape
    hkv = k_cache.shape[1]
    scale = d ** -0.5 if sm_scale is None else sm_scale
    ends = seq_lens.tolist()
    news = new_lens.tolist() if new_lens is not None else [tokens] * batch
    out = torch.zeros(q.shape, dtype=dtype, device=q.device)
    lse = torch.full(q.shape[:3], -math.inf, dtype=dtype, device=q.device)
    for b, (end, n) in enumerate(zip(ends, news)):
        if n == 0:
            continue
        k = kv8_values(k_cache, k_scale, block_table, b, end, dtype).repeat_interleave(hq // hkv, 0)
        v = kv8_values(v_cache, v_scale, block_table, b, end, dtype).repeat_interleave(hq // hkv, 0)
        for i in range(n):  # a row at a time: what it does not see stays out of its sums (0 * NaN would not)
            seen = end - n + i + 1
            s = torch.einsum("hd,hld->hl", q[b, i].to(dtype), k[:, :seen]) * scale
            lse[b, i] = torch.logsumexp(s, -1)
            out[b, i] = torch.einsum("hl,hld->hd", torch.softmax(s, -1), v[:, :seen])
    out = out if dtype == torch.float64 else out.to(q.dtype)
    return (out, lse) if return_lse else out
