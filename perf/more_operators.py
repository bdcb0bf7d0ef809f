"""Workloads for training the attention layers the token mixers serve: the norm of each query and key
head with the position rotation in the same pass (``qk_norm_rope``), its gradient
(``qk_norm_rope_bwd``), and the gradient of ``flash_attention_2`` (``flash_attention_2_bwd``).

``run`` computes a pass in plain torch operations (fp32) or, with ``own`` set, through the package's
plugin modules.  The definitions, shared by both:

* ``qk_norm_rope``: for every head row x of q and k, n = x / sqrt(mean(x^2) + eps) * weight (the queries'
  weight or the keys'); the 2 * half columns behind ``nope`` are then rotated in pairs (j, j + half) by
  the row of the cos and sin tables that the token's position names, y_j = n_j cos - n_{j+half} sin,
  y_{j+half} = n_j sin + n_{j+half} cos.  With several position axes (time, height, width) every pair
  takes the position of one axis: ``sections`` pairs for each axis, one axis after the other, or dealt
  out in turn (``interleaved``; pairs beyond an axis's share go to the first).
* ``qk_norm_rope_bwd``: the gradients of q, k and both weights from those of the outputs.
* ``flash_attention_2_bwd``: with P = exp(q k^T sm_scale - lse) under the causal mask (key j <= query i),
  delta = sum(do * o): dv = P^T do, dS = P * (do v^T - delta), dq = sm_scale dS k, dk = sm_scale dS^T q,
  dk and dv summed over the query heads that share a key/value head.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
THETA = 10000.0
# bounds of a drawn case: the largest listed norm's elements and the largest listed attention's operations
MOST_ROPE = 4 * 8192 * 40 * 128
MOST_FLOPS = 10 * 128 * 4 * 32 * (8192 * 8193 // 2)


def listed():
    return [
        # a decode step: one new token for each of 64 sequences, positions far apart, a quarter of the columns rotated
        dict(name="rope_decode", op="rope", B=64, S=1, Hq=16, Hkv=2, D=256, half=32, nope=0, axes=1, far=65536,
             inter=False, dtype="bf16", weight="bf16"),
        # two prompts with images: positions with three axes dealt out in turn, an odd length, fp16
        dict(name="rope_axes_fp16", op="rope", B=2, S=1031, Hq=8, Hkv=2, D=128, half=64, nope=0, axes=3, far=0,
             inter=True, dtype="fp16", weight="fp16"),
        # a batch of long prompts, whole heads rotated, positions in order
        dict(name="rope_prompts", op="rope", B=4, S=8192, Hq=32, Hkv=8, D=128, half=64, nope=0, axes=0, far=0,
             inter=False, dtype="bf16", weight="bf16"),
        # the gradient for a short sequence, one key head, fp16 with fp32 weights
        dict(name="rope_grad_short", op="rope_bwd", B=1, S=333, Hq=4, Hkv=1, D=64, half=16, nope=32, axes=1, far=512,
             inter=False, dtype="fp16", weight="fp32"),
        # the gradient for image prompts in 256-column heads, the last quarter rotated, three axes one after another
        dict(name="rope_grad_axes", op="rope_bwd", B=2, S=4096, Hq=16, Hkv=2, D=256, half=32, nope=192, axes=3, far=0,
             inter=False, dtype="bf16", weight="bf16"),
        # the gradient of the batch of long prompts
        dict(name="rope_grad_long", op="rope_bwd", B=4, S=8192, Hq=32, Hkv=8, D=128, half=64, nope=0, axes=0, far=0,
             inter=False, dtype="bf16", weight="bf16"),
        # the smallest attention gradient: a sequence just over a tile, grouped heads
        dict(name="attn_grad_short", op="attn", B=1, Sq=129, Skv=129, Hq=4, Hkv=2, D=128, causal=True, layout="bhsd"),
        # a short training batch in [batch, seq, heads, dim]
        dict(name="attn_grad_d64", op="attn", B=1, Sq=512, Skv=512, Hq=8, Hkv=8, D=64, causal=True, layout="bshd"),
        # attention to another sequence: no mask, lengths that differ and end inside tiles
        dict(name="attn_grad_cross", op="attn", B=3, Sq=1000, Skv=1531, Hq=12, Hkv=4, D=64, causal=False, layout="bshd"),
        # an ordinary training batch
        dict(name="attn_grad_batch", op="attn", B=8, Sq=2048, Skv=2048, Hq=8, Hkv=8, D=128, causal=True, layout="bhsd"),
        # 256-column heads, eight query heads to a key head
        dict(name="attn_grad_d256", op="attn", B=2, Sq=4096, Skv=4096, Hq=16, Hkv=2, D=256, causal=True, layout="bshd"),
        # long sequences, grouped heads
        dict(name="attn_grad_long", op="attn", B=4, Sq=8192, Skv=8192, Hq=32, Hkv=8, D=128, causal=True, layout="bhsd"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "rope_bwd", "attn", "attn"])
    d = rng.choice([64, 128, 256])
    hkv = rng.choice([1, 2, 3, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8])
    if op == "attn":
        causal = rng.random() < 0.7
        sq = _log(rng, 1, 8192)
        skv = sq if causal and rng.random() < 0.7 else _log(rng, 1, 8192)
        case = dict(op=op, B=1, Sq=sq, Skv=skv, Hq=hq, Hkv=hkv, D=d, causal=causal, layout=rng.choice(["bhsd", "bshd"]))
        case["B"] = _log(rng, 1, max(1, min(64, MOST_FLOPS // work(case)["flops"], 2 ** 28 // ((sq + skv) * hq * d))))
        while case["B"] == 1 and work(case)["flops"] > MOST_FLOPS:
            case["Sq"], case["Skv"] = case["Sq"] // 2, case["Skv"] // 2
        return case
    half = 8 * rng.randint(1, d // 16)
    most = MOST_ROPE // ((hq + hkv) * d)
    s = 1 if op == "rope" and rng.random() < 0.3 else _log(rng, 1, min(8192, most))
    return dict(op=op, B=_log(rng, 1, max(1, min(256, most // s))), S=s, Hq=hq, Hkv=hkv, D=d, half=half,
                nope=8 * rng.randint(0, (d - 2 * half) // 8), axes=rng.choice([0, 1, 2, 3]),
                far=s + _log(rng, 1, 65536), inter=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16"]),
                weight=rng.choice(["same", "fp32"]))


def _sections(case):
    """Pairs for each position axis: equal shares, the first axis takes what is left (None: one axis)."""
    if case["axes"] < 2:
        return None
    share = case["half"] // case["axes"]
    return (case["half"] - share * (case["axes"] - 1),) + (share,) * (case["axes"] - 1)


def _positions(case, gen):
    """[B, S] positions, [axes, B, S] where there are several, or None (the token's index)."""
    b, s, axes = case["B"], case["S"], case["axes"]
    if axes == 0:
        return None
    if axes == 1:  # a sequence's tokens follow one another from where its cached part ends
        start = torch.randint(0, max(1, case["far"] - s), (b, 1), generator=gen, device=DEV)
        return (start + torch.arange(s, device=DEV)).to(torch.int32)
    # patches of a grid of 32 columns between stretches of text, whose axes go together
    t = torch.arange(s, device=DEV).expand(b, s)
    text = (t // 256) % 2 == 0
    patch = t % 256
    grid = (t - patch + torch.zeros_like(t), t - patch + patch // 32, t - patch + patch % 32)
    shift = torch.randint(0, 7, (b, 1), generator=gen, device=DEV)
    return torch.stack([torch.where(text, t, g) + shift for g in grid[:axes]]).to(torch.int32)


def _table_rows(case):
    return max(case["far"], case["S"]) + 8


def _scores(s, b, h):
    """fp32 scores of the query heads that share key/value head h, [group, Sq, Skv]."""
    g = s["q"].shape[1] // s["k"].shape[1]
    x = s["q"][b, h * g:(h + 1) * g].float() @ s["k"][b, h].float().T * s["sm_scale"]
    if s["case"]["causal"]:
        x.masked_fill_(torch.ones(x.shape[1:], dtype=torch.bool, device=DEV).triu(1), -math.inf)
    return x


def _heads_first(s):
    """The state with its tensors [B, heads, S, D] (views)."""
    if s["case"]["layout"] == "bhsd":
        return s
    return {**s, **{n: s[n].transpose(1, 2) for n in ("do", "q", "k", "v", "o")}}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "attn":
        b, d, hq, hkv = case["B"], case["D"], case["Hq"], case["Hkv"]

        def normal(heads, length, norm):
            shape = (b, heads, length, d) if case["layout"] == "bhsd" else (b, length, heads, d)
            x = torch.randn(shape, generator=gen, device=DEV)
            if norm:  # queries and keys come out of their norm
                x = x / x.square().mean(-1, keepdim=True).sqrt()
            return x.to(torch.bfloat16)

        s = dict(case=case, sm_scale=d ** -0.5, q=normal(hq, case["Sq"], True), k=normal(hkv, case["Skv"], True),
                 v=normal(hkv, case["Skv"], False), do=normal(hq, case["Sq"], False) * 2.0 ** -6)
        s["o"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(b, hq, case["Sq"], dtype=torch.float32, device=DEV)
        t, g = _heads_first(s), hq // hkv
        for i in range(b):
            for h in range(hkv):
                x = _scores(t, i, h)
                s["lse"][i, h * g:(h + 1) * g] = torch.logsumexp(x, -1)
                t["o"][i, h * g:(h + 1) * g] = (torch.softmax(x, -1) @ t["v"][i, h].float()).to(torch.bfloat16)
        return s
    b, sl, hq, hkv, d = case["B"], case["S"], case["Hq"], case["Hkv"], case["D"]
    dt = DTYPES[case["dtype"]]
    wt = DTYPES.get(case["weight"], dt)
    heads = hq + 2 * hkv  # the projection's output, queries, keys and values side by side
    qkv = torch.randn(b, sl, heads, d, generator=gen, device=DEV)
    qkv = (qkv * torch.exp2(torch.randn(heads, 1, generator=gen, device=DEV))).to(dt)  # heads differ in size
    freq = THETA ** (-torch.arange(case["half"], dtype=torch.float64, device=DEV) / case["half"])
    angle = torch.arange(_table_rows(case), dtype=torch.float64, device=DEV)[:, None] * freq
    s = dict(case=case, q=qkv[:, :, :hq], k=qkv[:, :, hq:hq + hkv], cos=angle.cos().float(), sin=angle.sin().float(),
             q_weight=(1 + 0.2 * torch.randn(d, generator=gen, device=DEV)).to(wt),
             k_weight=(1 + 0.2 * torch.randn(d, generator=gen, device=DEV)).to(wt),
             positions=_positions(case, gen))
    if case["axes"] == 0:
        s["cos"], s["sin"] = s["cos"][:sl].contiguous(), s["sin"][:sl].contiguous()
    if case["op"] == "rope_bwd":
        s["dq"] = torch.randn(b, sl, hq, d, generator=gen, device=DEV).mul_(2.0 ** -4).to(dt)
        s["dk"] = torch.randn(b, sl, hkv, d, generator=gen, device=DEV).mul_(2.0 ** -4).to(dt)
    return s


# ------------------------------------------------------------------------------------ plain forms
def _pair_axis(case):
    """The position axis of every pair."""
    sections, half = _sections(case), case["half"]
    axis = torch.zeros(half, dtype=torch.long, device=DEV)
    at = sections[0] if sections else 0
    for a in range(1, case["axes"]):
        if case["inter"]:
            axis[a:a + case["axes"] * sections[a]:case["axes"]] = a
        else:
            axis[at:at + sections[a]] = a
            at += sections[a]
    return axis


def _plain_angles(s):
    """cos and sin of every token's pairs, [B or 1, S, 1, half]."""
    pos, case = s["positions"], s["case"]
    if pos is None:
        return s["cos"][None, :, None], s["sin"][None, :, None]
    if pos.ndim == 2:
        row = pos.long()
        return s["cos"][row][:, :, None], s["sin"][row][:, :, None]
    row = pos.long()[_pair_axis(case)].permute(1, 2, 0)                                  # [B, S, half]
    pair = torch.arange(case["half"], device=DEV)
    return s["cos"][row, pair][:, :, None], s["sin"][row, pair][:, :, None]


def _plain_rotate(case, n, c, sn):
    lo, mid = case["nope"], case["nope"] + case["half"]
    hi = mid + case["half"]
    x0, x1 = n[..., lo:mid], n[..., mid:hi]
    return torch.cat((n[..., :lo], x0 * c - x1 * sn, x0 * sn + x1 * c, n[..., hi:]), -1)


def _plain_rope(s):
    c, sn = _plain_angles(s)
    out = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        xf = x.float()
        n = xf / (xf.square().mean(-1, keepdim=True) + EPS).sqrt() * w.float()
        out.append(_plain_rotate(s["case"], n, c, sn).to(x.dtype))
    return out


def _plain_rope_bwd(s):
    c, sn = _plain_angles(s)
    grads, weights = [], []
    for dy, x, w in ((s["dq"], s["q"], s["q_weight"]), (s["dk"], s["k"], s["k_weight"])):
        xf, wf = x.float(), w.float()
        inv = 1 / (xf.square().mean(-1, keepdim=True) + EPS).sqrt()
        g = _plain_rotate(s["case"], dy.float(), c, -sn)                                  # the rotation's transpose
        weights.append((g * xf * inv).double().sum((0, 1, 2)).to(w.dtype))                # long sums
        gw = g * wf
        grads.append((inv * (gw - xf * inv * inv * (gw * xf).mean(-1, keepdim=True))).to(x.dtype))
    return grads + weights


def _plain_attn(s):
    t = _heads_first(s)
    out = [torch.empty_like(s[n]) for n in ("q", "k", "v")]
    dq, dk, dv = (x if s["case"]["layout"] == "bhsd" else x.transpose(1, 2) for x in out)
    b, hkv = t["k"].shape[:2]
    g = t["q"].shape[1] // hkv
    for i in range(b):
        for h in range(hkv):
            hs = slice(h * g, (h + 1) * g)
            q, do, k, v = t["q"][i, hs].float(), t["do"][i, hs].float(), t["k"][i, h].float(), t["v"][i, h].float()
            p = torch.exp(_scores(t, i, h) - t["lse"][i, hs, :, None])
            dv[i, h] = (p.flatten(0, 1).T @ do.flatten(0, 1)).to(torch.bfloat16)
            delta = (do * t["o"][i, hs].float()).sum(-1, keepdim=True)
            ds = p * (do @ v.T - delta) * s["sm_scale"]
            dq[i, hs] = (ds @ k).to(torch.bfloat16)
            dk[i, h] = (ds.flatten(0, 1).T @ q.flatten(0, 1)).to(torch.bfloat16)
    return out


# ------------------------------------------------------------------------------------ the package's calls
def _own(s):
    from kernel_opt_agent_b200 import flash_attention_2_bwd, qk_norm_rope, qk_norm_rope_bwd

    case = s["case"]
    if case["op"] == "attn":
        return flash_attention_2_bwd.kernel_fn(s["do"], s["q"], s["k"], s["v"], s["o"], s["lse"], case["causal"],
                                               s["sm_scale"], layout=case["layout"])
    args = (s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"])
    kw = dict(eps=EPS, nope_dim=case["nope"], sections=_sections(case), interleaved=case["axes"] > 1 and case["inter"])
    if case["op"] == "rope":
        return qk_norm_rope.kernel_fn(*args, **kw)
    return qk_norm_rope_bwd.kernel_fn(s["dq"], s["dk"], *args, **kw)


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "rope_bwd": _plain_rope_bwd, "attn": _plain_attn}[state["case"]["op"]](state)


def work(case):
    b, d, hq, hkv = case["B"], case["D"], case["Hq"], case["Hkv"]
    if case["op"] == "attn":
        sq, skv = case["Sq"], case["Skv"]
        pairs = sq * skv
        if case["causal"]:
            n = min(sq, skv)
            pairs = n * (n + 1) // 2 + (sq - n) * skv
        # q, o, do read and dq written; k, v read and dk, dv written; lse read
        return {"bytes": b * (4 * hq * sq * d * 2 + 4 * hkv * skv * d * 2 + hq * sq * 4), "flops": 10 * b * hq * pairs * d}
    rows = b * case["S"]
    small = 2 if case["weight"] != "fp32" else 4
    axes = case["axes"]
    used = case["S"] if axes == 0 else min(_table_rows(case), rows)                       # table rows that a call needs
    tables = used * case["half"] * 2 * 4 + axes * rows * 4
    elements = rows * (hq + hkv) * d
    if case["op"] == "rope":
        return {"bytes": elements * 2 * 2 + tables + 2 * d * small, "flops": 8 * elements}
    return {"bytes": elements * 2 * 3 + tables + 4 * d * small, "flops": 16 * elements}


# ------------------------------------------------------------------------------------ in 64 bits
def _exact_turns(case, s):
    """exp(i angle) of every token's pairs as the tables hold it, complex128 [B, S, 1, half]."""
    table = torch.complex(s["cos"].double(), s["sin"].double())
    pos, (b, sl) = s["positions"], (case["B"], case["S"])
    if pos is None:
        return table[:sl].expand(b, sl, -1)[:, :, None]
    if pos.ndim == 2:
        return table[pos.long()][:, :, None]
    sections, axes, cols = _sections(case), case["axes"], []
    bounds = [sum(sections[:a + 1]) for a in range(axes)]
    for j in range(case["half"]):
        if case["inter"]:
            a = j % axes if j < axes * sections[j % axes] else 0
        else:
            a = sum(j >= e for e in bounds)
        cols.append(table[pos[a].long(), j])
    return torch.stack(cols, -1)[:, :, None]


def _exact_forward(case, x, w, turns):
    n = w * x * torch.rsqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)
    half, nope = case["half"], case["nope"]
    z = torch.complex(n[..., nope:nope + half], n[..., nope + half:nope + 2 * half]) * turns
    return torch.cat((n[..., :nope], z.real, z.imag, n[..., nope + 2 * half:]), -1)


def _exact_rope(case, s):
    turns = _exact_turns(case, s)
    return [_exact_forward(case, s[n].double(), s[n + "_weight"].double(), turns) for n in ("q", "k")]


def _exact_rope_bwd(case, s):
    turns = _exact_turns(case, s)
    grads, weights = [], []
    for n in ("q", "k"):
        w = s[n + "_weight"].double().requires_grad_()
        dx, dw = torch.empty(s[n].shape, dtype=torch.float64, device=DEV), 0
        for i in range(case["B"]):  # a sequence at a time
            x = s[n][i:i + 1].double().requires_grad_()
            gx, gw = torch.autograd.grad(_exact_forward(case, x, w, turns[i:i + 1]), (x, w), s["d" + n][i:i + 1].double())
            dx[i], dw = gx[0], dw + gw
        grads.append(dx)
        weights.append(dw)
    return grads + weights


def _exact_attn(case, s):
    t = _heads_first(s)
    b, hq, sq, d = t["q"].shape
    g = hq // t["k"].shape[1]
    dq = torch.zeros(t["q"].shape, dtype=torch.float64, device=DEV)
    dk, dv = (torch.zeros(t["k"].shape, dtype=torch.float64, device=DEV) for _ in range(2))
    for i in range(b):
        for h in range(hq):
            for lo in range(0, sq, 2048):  # a block of queries at a time, the keys that it sees
                hi = min(sq, lo + 2048)
                end = min(hi, case["Skv"]) if case["causal"] else case["Skv"]
                q, do, o = (t[n][i, h, lo:hi].double() for n in ("q", "do", "o"))
                k, v = (t[n][i, h // g, :end].double() for n in ("k", "v"))
                w = torch.exp(torch.einsum("qd,kd->qk", q, k) * s["sm_scale"] - t["lse"][i, h, lo:hi, None].double())
                if case["causal"]:
                    rows = torch.arange(lo, hi, device=DEV)[:, None]
                    w = torch.where(torch.arange(end, device=DEV) <= rows, w, 0.0)
                dv[i, h // g, :end] += torch.einsum("qk,qd->kd", w, do)
                w *= torch.einsum("qd,kd->qk", do, v) - torch.einsum("qd,qd->q", do, o)[:, None]
                dq[i, h, lo:hi] = torch.einsum("qk,kd->qd", w, k) * s["sm_scale"]
                dk[i, h // g, :end] += torch.einsum("qk,qd->kd", w, q) * s["sm_scale"]
    return [dq, dk, dv] if case["layout"] == "bhsd" else [x.transpose(1, 2) for x in (dq, dk, dv)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "rope_bwd": _exact_rope_bwd, "attn": _exact_attn}[case["op"]](case, s)
