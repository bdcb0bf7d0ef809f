"""Workloads for the serving-step operators around the token mixers: the residual + RMS norm that
writes FP8 (``add_rms_norm_quant``), the paged 8-bit key/value cache (``kv8_append``) and the
attention that reads it (``kv8_attention``).

``run`` computes a pass in plain torch operations (fp32) or, with ``own`` set, through the
package's plugin modules.  The definitions, shared by both:

* ``add_rms_norm_quant``: h = T(x + residual) (T: the inputs' type), u = h * weight,
  inv_rms = 1 / sqrt(mean(h^2) + eps); for every group of columns a = max(max |u|, 2^-100),
  y = e4m3(u * (448 / a)), scale = a * inv_rms / 448.  y * scale is the normalised row.
* ``kv8_append``: tokens enter pages of a cache held in 8 bits with one scale per (page, head),
  for keys and values apart.  A scale is the smallest power of two (at least 2^-100) with
  max |x| <= qmax * scale over the page's tokens (qmax 448 for e4m3, 127 for int8); where new tokens
  raise the scale of a page, its older tokens are rounded again to the new one.
* ``kv8_attention``: query i of the T newest tokens of a sequence attends to every cached token up to
  its own position, o = softmax(q k^T sm_scale) v with k, v the values the cache stands for.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}
TINY = 2.0 ** -100
EPS = 1e-6
# bounds of a drawn attention: cached keys, and operations of about the largest listed case
MOST_CACHE = 16 * 65536 * 2 * 256
MOST_FLOPS = 10_000_000_000


def listed():
    return [
        # one token of one sequence enters a layer: nothing but latency
        dict(name="norm_token", op="norm", M=1, N=4096, group=128, dtype="bf16"),
        # a ragged batch of short rows, one scale per row, fp16
        dict(name="norm_rows_fp16", op="norm", M=1023, N=768, group=0, dtype="fp16"),
        # a prefill chunk, a scale per 32 columns
        dict(name="norm_chunk_g32", op="norm", M=2048, N=5120, group=32, dtype="bf16"),
        # a long prompt through a wide layer, a scale per 128 columns
        dict(name="norm_prompt", op="norm", M=4096, N=7168, group=128, dtype="bf16"),
        # a decode step of 64 sequences: one token each, pages partly filled
        dict(name="append_token", op="append", B=64, T=1, L=4096, Hkv=2, D=256, page=64, cache="e4m3", dtype="bf16"),
        # ragged chunks of up to 333 tokens behind shorter prefixes, small pages, int8
        dict(name="append_chunk_int8", op="append", B=7, T=333, L=1031, Hkv=4, D=64, page=16, cache="int8",
             dtype="fp16"),
        # whole prompts of up to 8192 tokens
        dict(name="append_prompt", op="append", B=4, T=8192, L=8192, Hkv=8, D=128, page=64, cache="e4m3",
             dtype="bf16"),
        # one short sequence: latency
        dict(name="attn_short", op="attn", B=1, T=1, L=129, Hq=16, Hkv=2, D=256, page=16, cache="e4m3",
             dtype="bf16"),
        # verification of four drafted tokens per sequence, plain multi-head attention, int8
        dict(name="attn_verify_int8", op="attn", B=16, T=4, L=1031, Hq=8, Hkv=8, D=64, page=32, cache="int8",
             dtype="fp16"),
        # a decode batch of mixed lengths, grouped-query heads
        dict(name="attn_batch", op="attn", B=64, T=1, L=4096, Hq=32, Hkv=8, D=128, page=64, cache="e4m3",
             dtype="bf16"),
        # one long sequence: few heads, the work lies along the sequence
        dict(name="attn_long", op="attn", B=1, T=1, L=65536, Hq=16, Hkv=2, D=256, page=64, cache="e4m3",
             dtype="bf16"),
        # long sequences of mixed lengths
        dict(name="attn_long_batch", op="attn", B=16, T=1, L=65536, Hq=16, Hkv=2, D=256, page=128, cache="e4m3",
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "append", "attn"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "norm":
        n = 128 * _log(rng, 1, 96)
        return dict(op=op, M=_log(rng, 1, min(8192, 4096 * 7168 // n)), N=n, group=rng.choice([0, 32, 128]),
                    dtype=dtype)
    d = rng.choice([64, 128, 256])
    hkv = rng.choice([1, 2, 3, 4, 8])
    page, cache = rng.choice([16, 32, 64, 128]), rng.choice(["e4m3", "int8"])
    if op == "append":
        most = 4 * 8192 * 8 * 128 // (hkv * d)  # tokens of the largest listed append
        t = _log(rng, 1, 8192)
        b = _log(rng, 1, max(1, min(128, most // t)))
        return dict(op=op, B=b, T=t, L=t + _log(rng, 1, 4096), Hkv=hkv, D=d, page=page, cache=cache, dtype=dtype)
    hq = hkv * rng.choice([1, 2, 4, 5, 7, 8, 12])
    t = rng.choice([1, 1, 1, 2, 3, 5, 8])
    length = _log(rng, t, min(65536, MOST_FLOPS // (4 * hq * d * t)))
    most = min(128, MOST_CACHE // (2 * length * hkv * d), MOST_FLOPS // (4 * hq * d * t * length))
    return dict(op=op, B=_log(rng, 1, max(1, most)), T=t, L=length, Hq=hq, Hkv=hkv, D=d, page=page, cache=cache,
                dtype=dtype)


def _lens(case):
    """(seq_lens, new_lens) of a batch: lengths spread over [L/4, L] with one of L itself, an empty
    sequence in every larger batch; chunks of several tokens are ragged."""
    b, t, length = case["B"], case["T"], case["L"]
    rng = random.Random("%d %d %d %d %d" % (b, t, length, case["Hkv"], case["D"]))
    seq = [length] + [rng.randint(max(t, length // 4), length) for _ in range(b - 1)]
    new = [t] + [t if case["op"] == "attn" or t == 1 else rng.randint(1, t) for _ in range(b - 1)]
    if b > 4:
        seq[b // 2], new[b // 2] = 0, 0
    return seq, new


def _pow2_scale(amax, cache):
    """The smallest power of two s >= 2^-100 with amax <= qmax * s (exact: by exponent and mantissa)."""
    bits, limit = (9, 0.875) if cache == "e4m3" else (7, 0.9921875)  # 448 = 0.875 * 2^9, 127 = 0.9921875 * 2^7
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - bits + (m > limit), -100).clamp_min(-100)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _to8(x, cache):
    """x / scale (already divided) rounded to the cache's type: nearest, ties to even."""
    return x.to(torch.float8_e4m3fn) if cache == "e4m3" else x.round().to(torch.int8)


def _make_cache(gen, pages, case):
    """A filled cache [pages, Hkv, page, D] and its scales: N(0,1) values whose channels differ in size."""
    hkv, page, d, cache = case["Hkv"], case["page"], case["D"], case["cache"]
    vals = torch.empty(pages, hkv, page, d, dtype=DTYPES[cache], device=DEV)
    scales = torch.empty(pages, hkv, dtype=torch.float32, device=DEV)
    channel = torch.exp2(torch.randn(hkv, 1, d, generator=gen, device=DEV) * 0.5)
    step = max(1, (1 << 28) // (hkv * page * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = torch.randn(n, hkv, page, d, generator=gen, device=DEV) * channel
        scales[p:p + n] = _pow2_scale(x.abs().amax((2, 3)), cache)
        vals[p:p + n] = _to8(x / scales[p:p + n, :, None, None], cache)
    return vals, scales


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        m, n = case["M"], case["N"]
        x = torch.randn(m, n, generator=gen, device=DEV)
        res = torch.randn(m, n, generator=gen, device=DEV) * 4  # the residual stream outgrows its updates
        w = 1 + 0.2 * torch.randn(n, generator=gen, device=DEV)
        return dict(case=case, x=x.to(dt), residual=res.to(dt), weight=w.to(dt))
    b, t, hkv, d, page = case["B"], case["T"], case["Hkv"], case["D"], case["page"]
    seq, new = _lens(case)
    per = -(-max(seq) // page)
    need = [-(-s // page) for s in seq]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros(b, per, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s = dict(case=case, block_table=table, seq_lens=torch.tensor(seq, dtype=torch.int32, device=DEV),
             new_lens=torch.tensor(new, dtype=torch.int32, device=DEV))
    s["k_cache"], s["k_scale"] = _make_cache(gen, pages, case)
    s["v_cache"], s["v_scale"] = _make_cache(gen, pages, case)
    if case["op"] == "append":
        s["k"] = torch.randn(b, t, hkv, d, generator=gen, device=DEV).to(dt)
        s["v"] = torch.randn(b, t, hkv, d, generator=gen, device=DEV).to(dt)
    else:
        s["q"] = (2 * torch.randn(b, t, case["Hq"], d, generator=gen, device=DEV)).to(dt)
    return s


# ------------------------------------------------------------------------------------ plain forms
def _plain_norm(s):
    case = s["case"]
    h = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    hf = h.float()
    inv_rms = 1 / (hf.square().mean(-1, keepdim=True) + EPS).sqrt()
    m, n = hf.shape
    group = case["group"] or n
    u = (hf * s["weight"].float()).view(m, n // group, group)
    a = u.abs().amax(-1).clamp_min(TINY)
    y = (u * (torch.full_like(a, 448.0) / a).unsqueeze(-1)).to(torch.float8_e4m3fn).view(m, n)
    scale = a * inv_rms / torch.full_like(a, 448.0)
    return [y, scale.t().contiguous() if case["group"] else scale.view(m), h]


def _plain_append_one(s, x, vals, scales):
    case = s["case"]
    page, cache, t = case["page"], case["cache"], case["T"]
    start = s["seq_lens"] - s["new_lens"]
    touched = 1 if t == 1 else (t - 1) // page + 2
    pj = start[:, None] // page + torch.arange(touched, device=DEV)                       # [B, J] page index
    pos = pj[:, :, None] * page + torch.arange(page, device=DEV)                          # [B, J, page]
    is_new = (pos >= start[:, None, None]) & (pos < s["seq_lens"][:, None, None])
    b, j = is_new.any(-1).nonzero(as_tuple=True)                                          # pages that change
    pos, is_new, first = pos[b, j], is_new[b, j], start[b]
    ids = s["block_table"][b, pj[b, j]].long()
    new = x[b[:, None], (pos - first[:, None]).clamp(0, t - 1)].float().transpose(1, 2)   # [n, Hkv, page, D]
    mask = is_new[:, None, :, None]
    amax = torch.where(mask, new.abs(), 0.0).amax((2, 3))
    has_old = (pos[:, 0] < first)[:, None]
    old_scale = scales[ids]
    scale = torch.maximum(_pow2_scale(amax, cache), torch.where(has_old, old_scale, 0.0))
    raw = vals.view(torch.uint8)[ids].view(vals.dtype)
    again = _to8(raw.float() * (old_scale / scale)[:, :, None, None], cache)
    is_old = (pos < first[:, None])[:, None, :, None]
    put = torch.where(mask, _to8(new / scale[:, :, None, None], cache).view(torch.uint8),
                      torch.where(is_old, again.view(torch.uint8), raw.view(torch.uint8)))
    vals.view(torch.uint8)[ids] = put
    scales[ids] = scale


def _plain_append(s):
    _plain_append_one(s, s["k"], s["k_cache"], s["k_scale"])
    _plain_append_one(s, s["v"], s["v_cache"], s["v_scale"])
    return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]


def _gathered(s, vals, scales):
    """The cached values of every sequence in order, fp32 [B, Hkv, pages * page, D]."""
    ids = s["block_table"].long()
    x = vals.view(torch.uint8)[ids].view(vals.dtype).float() * scales[ids][..., None, None]
    b, p, hkv, page, d = x.shape
    return x.transpose(1, 2).reshape(b, hkv, p * page, d)


def _plain_attn(s):
    case, q = s["case"], s["q"]
    b, t, hq, d = q.shape
    hkv = case["Hkv"]
    k = _gathered(s, s["k_cache"], s["k_scale"])
    qr = q.float().view(b, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    score = qr @ k.transpose(2, 3) * d ** -0.5
    del k
    last = (s["seq_lens"] - s["new_lens"])[:, None] + torch.arange(t, device=DEV)         # a query's position
    last = torch.where(torch.arange(t, device=DEV) < s["new_lens"][:, None], last, -1)
    seen = torch.arange(score.shape[-1], device=DEV) <= last[:, :, None]                  # [B, T, L]
    seen = seen.repeat_interleave(hq // hkv, 1)[:, None]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    o = (p @ _gathered(s, s["v_cache"], s["v_scale"])) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.view(b, hkv, t, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d).to(q.dtype)


# ------------------------------------------------------------------------------------ the package's calls
def _own(s):
    from kernel_opt_agent_b200 import add_rms_norm_quant, kv8_append, kv8_attention

    case = s["case"]
    if case["op"] == "norm":
        return add_rms_norm_quant.kernel_fn(s["x"], s["residual"], s["weight"], EPS, group=case["group"] or None)
    if case["op"] == "append":
        return kv8_append.kernel_fn(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                                    s["block_table"], s["seq_lens"], s["new_lens"])
    return kv8_attention.kernel_fn(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"],
                                   s["seq_lens"], s["new_lens"])


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "append": _plain_append, "attn": _plain_attn}[state["case"]["op"]](state)


def work(case):
    if case["op"] == "norm":
        m, n = case["M"], case["N"]
        groups = n // case["group"] if case["group"] else 1
        return {"bytes": m * n * (2 + 2 + 2 + 1) + n * 2 + m * groups * 4, "flops": 7 * m * n}
    seq, new = _lens(case)
    hkv, d, page = case["Hkv"], case["D"], case["page"]
    if case["op"] == "append":
        pages = sum((s - 1) // page - (s - n) // page + 1 for s, n in zip(seq, new) if n)
        return {"bytes": 2 * (sum(new) * hkv * d * 3 + pages * hkv * 4), "flops": 2 * 2 * sum(new) * hkv * d}
    pages = sum(-(-s // page) for s in seq)
    io = sum(new) * case["Hq"] * d * 2 * 2
    return {"bytes": 2 * (sum(seq) * hkv * d + pages * hkv * 4) + pages * 4 + io,
            "flops": 4 * case["Hq"] * d * sum(n * s - n * (n - 1) // 2 for s, n in zip(seq, new))}


# ------------------------------------------------------------------------------------ in 64 bits

def _round_e4m3(x):
    """The nearest e4m3 value of each |x| <= 448 (and a little over), ties to even."""
    a = x.abs().clamp_max(448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))).clamp(-6, 8) - 3)
    r = torch.round(a / step) * step
    return torch.copysign(r, x)


def _exact_norm(case, s):
    h = (s["x"].double() + s["residual"].double()).to(s["x"].dtype).double()
    n = h.shape[1]
    group = case["group"] or n
    u = (h * s["weight"].double()).unflatten(1, (n // group, group))
    a = torch.clamp(u.abs().max(-1).values, min=TINY)
    y = _round_e4m3(448.0 * u / a[..., None]).flatten(1)
    scale = a / 448.0 * torch.rsqrt((h * h).sum(-1, keepdim=True) / n + EPS)
    return [y, scale.T if case["group"] else scale[:, 0], h]


def _exact_append(case, s):
    page, e4m3 = case["page"], case["cache"] == "e4m3"
    outs = []
    seq, new = _lens(case)
    table = s["block_table"].tolist()
    for name in ("k", "v"):
        vals = s[name + "_cache"].double()
        scales = s[name + "_scale"].double()
        old_scales = scales.tolist()
        found = []
        for b, (end, n) in enumerate(zip(seq, new)):
            for p in range((end - n) // page, (end - 1) // page + 1 if n else 0):
                lo, hi = max(end - n, p * page), min(end, (p + 1) * page)
                x = s[name][b, lo - end + n:hi - end + n].double().transpose(0, 1)  # [Hkv, tokens, D]
                found.append((table[b][p], lo - p * page, hi - p * page, x, x.abs().amax((1, 2))))
        tops = torch.stack([f[4] for f in found]).tolist()
        for (pid, lo, hi, x, _), top in zip(found, tops):
            per_head = []
            for h, t in enumerate(top):
                e = -100
                if t > 0:
                    e = max(e, math.ceil(math.log2(t / QMAX[case["cache"]])))
                    while t > QMAX[case["cache"]] * 2.0 ** e:
                        e += 1
                    while e > -100 and t <= QMAX[case["cache"]] * 2.0 ** (e - 1):
                        e -= 1
                per_head.append(max(2.0 ** e, old_scales[pid][h] if lo > 0 else 0.0))
            grown = [o != g for o, g in zip(old_scales[pid], per_head)]
            to = torch.tensor(per_head, dtype=torch.float64, device=DEV)[:, None, None]
            rnd = _round_e4m3 if e4m3 else torch.round
            vals[pid, :, lo:hi] = rnd(x / to)
            if lo > 0 and any(grown):
                was = torch.tensor(old_scales[pid], dtype=torch.float64, device=DEV)[:, None, None]
                vals[pid, :, :lo] = rnd(vals[pid, :, :lo] * was / to)
            scales[pid] = to[:, 0, 0]
        outs.append((vals if e4m3 else None, scales))
    return [outs[0][0], outs[1][0], outs[0][1], outs[1][1]]


def _exact_attn(case, s):
    seq, new = _lens(case)
    hkv, d, page = case["Hkv"], case["D"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, (end, n) in enumerate(zip(seq, new)):
        if not end:
            continue
        ids = s["block_table"][b, :-(-end // page)].long()
        for h in range(hkv):
            k, v = ((s[c + "_cache"][:, h].view(torch.uint8)[ids].view(s[c + "_cache"].dtype).double()
                     * s[c + "_scale"][ids, h].double()[:, None, None]).flatten(0, 1)[:end] for c in "kv")
            g = case["Hq"] // hkv
            for i in range(n):
                w = torch.softmax(s["q"][b, i, h * g:(h + 1) * g].double() @ k[:end - n + i + 1].T / math.sqrt(d), -1)
                out[b, i, h * g:(h + 1) * g] = w @ v[:end - n + i + 1]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "attn": _exact_attn}[case["op"]](case, s)
