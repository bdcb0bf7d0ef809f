"""The attention's gradients in the 2-norm, by blocks of 128 rows, up to the longest of the config sizes: an element's own bound
grows with the number of terms in its sum, a lost step of 128 queries and keys shows in the norm of its blocks.

Bound.  An output is a sum of terms t, each with an operand (P or dS) rounded to bf16: off by at most 2^-8 |t|, with independent
signs, so the error's square is, on the mean, at most 2^-16 sum t^2 (a third of that for errors spread evenly over
the step).  Behind that the result is rounded, 2^-8 of itself.  Over a block the norm of the error is therefore at most
2^-8 (R + N), R the root of the sum of all squared terms and N the norm of the result; the third leaves room for a block
that is not the mean, and for fp32's own errors, 2^-20 of the terms.  In numbers this is about 0.008 of N.  A step lost, one
of n of a block's, is about 1 / sqrt(n) of N; the most here are 4 heads x 33 tiles: 0.087."""

import pytest
import torch

from kernel_opt_agent_b200 import flash_attention_2 as fa2
from kernel_opt_agent_b200 import flash_attention_2_bwd as bwd
from kernel_opt_agent_b200.kernel_configs import KERNEL_CONFIGS

CONFIG = KERNEL_CONFIGS["flash_attention_2_bwd"]


def gradients(do, q, k, v, o, lse, causal, scale, group):
    """fp32 gradients of one key/value head's query heads [group, S, D], and the roots of their terms' summed squares."""
    do, q, k, v, o = (t.float() for t in (do, q, k, v, o))
    p = torch.exp(q @ k.T * scale - lse[..., None])
    if causal:
        p = p.masked_fill(torch.ones(p.shape[1:], dtype=torch.bool, device=p.device).triu(1), 0.0)
    ds = p * (do @ v.T - (do * o).sum(-1, keepdim=True)) * scale

    def both(a, b):
        return a @ b, (a.square() @ b.square()).sqrt()

    flat = lambda t: t.flatten(0, 1)  # noqa: E731
    return both(ds, k), both(flat(ds).T, flat(q)), both(flat(p).T, flat(do))


def block_norms(x):
    """Norms of blocks of 128 rows, the last of what is left: [..., S, D] -> [..., blocks]."""
    return torch.stack([b.double().square().sum((-1, -2)).sqrt() for b in x.split(128, -2)], -1)


def worst_blocks(got, do, q, k, v, o, lse, causal, scale, layout):
    """The most that a block's error takes of its bound, for dq, dk and dv."""
    first = (lambda t: t) if layout == "bhsd" else (lambda t: t.transpose(1, 2))
    do, q, k, v, o = (first(t) for t in (do, q, k, v, o))
    got = [first(t) for t in got]
    group = q.shape[1] // k.shape[1]
    worst = [0.0, 0.0, 0.0]
    for b in range(q.shape[0]):
        for h in range(k.shape[1]):
            hs = slice(h * group, (h + 1) * group)
            want = gradients(do[b, hs], q[b, hs], k[b, h], v[b, h], o[b, hs], lse[b, hs], causal, scale, group)
            for n, (x, (ref, root)) in enumerate(zip((got[0][b, hs], got[1][b, h], got[2][b, h]), want)):
                bound = 2.0 ** -8 * (block_norms(root) + block_norms(ref)) + 2.0 ** -100
                worst[n] = max(worst[n], (block_norms(x.float() - ref) / bound).max().item())
    return worst


def check(do, q, k, v, o, lse, causal, sm_scale, layout="bhsd"):
    got = bwd.kernel_fn(do, q, k, v, o, lse, causal, sm_scale, layout=layout)
    bwd.check_device_status(q.device)
    worst = worst_blocks(got, do, q, k, v, o, lse, causal, sm_scale, layout)
    assert max(worst) <= 1.0, worst


@pytest.mark.gpu
@pytest.mark.parametrize("label,size", CONFIG["test_sizes"] + CONFIG["edge_sizes"],
                         ids=[label for label, _ in CONFIG["test_sizes"] + CONFIG["edge_sizes"]])
def test_blocks_at_the_config_sizes(cuda_device, label, size):
    check(**CONFIG["input_generator"](size, torch.bfloat16, "cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("b,hq,hkv,sq,skv,d,causal,layout", [
    (1, 8, 2, 4099, 4099, 64, True, "bshd"), (1, 8, 2, 4097, 4097, 256, True, "bhsd"), (2, 3, 3, 2500, 4100, 64, False, "bhsd"),
    (1, 4, 1, 4100, 2500, 128, False, "bshd"), (1, 2, 1, 1000, 3900, 256, False, "bshd"), (1, 2, 2, 4000, 1000, 256, True, "bhsd"),
    (4, 8, 4, 1500, 1500, 128, False, "bhsd"), (40, 1, 1, 300, 300, 64, True, "bhsd"), (40, 4, 4, 130, 600, 128, False, "bhsd")])
def test_blocks_at_long_and_ragged_sizes(cuda_device, b, hq, hkv, sq, skv, d, causal, layout):
    gen = torch.Generator().manual_seed(sq + skv)

    def t(h, s):
        return torch.randn((b, h, s, d) if layout == "bhsd" else (b, s, h, d), generator=gen).to(torch.bfloat16).cuda()

    q, k, v, do = t(hq, sq), t(hkv, skv), t(hkv, skv), t(hq, sq)
    o, lse = fa2.kernel_fn(q, k, v, causal, layout=layout, return_lse=True)
    check(do, q, k, v, o, lse, causal, d ** -0.5, layout)


def test_the_bound_notices_a_lost_step():
    """On the CPU, in the oracle: the bound holds for rounded operands and is passed where one step of 128 x 128 is left out."""
    gen = torch.Generator().manual_seed(0)
    s, d, group, scale = 1536, 64, 2, 0.125
    q, do, k, v = (torch.randn(*n, s, d, generator=gen).to(torch.bfloat16) for n in ((group,), (group,), (), ()))
    mask = torch.ones(s, s, dtype=torch.bool).triu(1)
    x = (q.float() @ k.float().T * scale).masked_fill(mask, float("-inf"))
    lse, o = torch.logsumexp(x, -1), (torch.softmax(x, -1) @ v.float()).to(torch.bfloat16)
    p = torch.exp(x - lse[..., None])
    ds = p * (do.float() @ v.float().T - (do.float() * o.float()).sum(-1, keepdim=True))

    def results(lost):
        r = lambda t: t.to(torch.bfloat16).float()  # noqa: E731
        pr, dr = r(p), r(ds)
        if lost is not None:
            h, i, j = lost
            pr[h, i * 128:(i + 1) * 128, j * 128:(j + 1) * 128] = 0
            dr[h, i * 128:(i + 1) * 128, j * 128:(j + 1) * 128] = 0
        flat = lambda t: t.flatten(0, 1)  # noqa: E731
        out = ((dr * scale) @ k.float(), flat(dr * scale).T @ flat(q.float()), flat(pr).T @ flat(do.float()))
        return [t.to(torch.bfloat16)[None] for t in (out[0], out[1][None], out[2][None])]

    args = (do[None], q[None], k[None, None], v[None, None], o[None], lse[None], True, scale, "bhsd")
    assert max(worst_blocks(results(None), *args)) <= 1.0
    for lost in ((0, 0, 0), (1, 5, 2), (0, 11, 0), (1, 11, 11), (0, 11, 7)):
        assert min(worst_blocks(results(lost), *args)) > 1.0, lost
