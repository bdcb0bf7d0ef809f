"""The attention's gradients on a B200 against the formula in 64 bits.

Tolerances.  Operands are bf16; P and dS are rounded to bf16 once more (at most half a step, 2^-8 of
the value), products are accumulated in fp32 and the results rounded to bf16 (2^-8 of the value).  An
output is a sum of terms t_i, each off by at most 2^-8 |t_i| (its P or dS rounding), so it is off by at most
2^-8 sum |t_i| plus its own rounding: the test compares against that bound, formed in 64 bits from the
absolute values.  dS is P (dP - delta), where dP and delta carry fp32 errors of at most (d + 8) 2^-24 of
their absolute sums, which the bound adds, as it does P's: the exponent c s - lse in fp32 is off by a few
2^-24 of its parts and of the absolute sum behind s.
"""

import math

import pytest
import torch

from kernel_opt_agent_b200 import flash_attention_2 as fa2
from kernel_opt_agent_b200 import flash_attention_2_bwd as bwd

pytestmark = pytest.mark.gpu


def formula(do, q, k, v, o, lse, causal, sm_scale, layout):
    """(dq, dk, dv) and bounds of their errors, float64, in the inputs' layout."""
    if layout == "bshd":
        do, q, k, v, o = (t.transpose(1, 2) for t in (do, q, k, v, o))
    do, q, k, v, o, lse = (t.double() for t in (do, q, k, v, o, lse))
    g = q.shape[1] // k.shape[1]
    kx, vx = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = q @ kx.transpose(2, 3) * sm_scale
    seen = torch.ones(s.shape[2:], dtype=torch.bool, device=s.device)
    if causal:
        seen = seen.tril()
    p = torch.where(seen, torch.exp(s - lse[..., None]), 0.0)
    dp = do @ vx.transpose(2, 3)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    d = q.shape[-1]
    # relative error of P before its rounding: the exponent's, in fp32
    s_abs = (q.abs() @ kx.abs().transpose(2, 3)) * sm_scale
    rel_p = (s_abs + s.abs() + lse.abs()[..., None]) * (d / 16 + 8) * 2.0 ** -24 + 2.0 ** -21
    dp_err = ((do.abs() @ vx.abs().transpose(2, 3)) + (do.abs() * o.abs()).sum(-1, keepdim=True)) * (d + 8) * 2.0 ** -24
    p_err = p * (rel_p + 2.0 ** -8)
    ds_err = ds.abs() * (rel_p + 2.0 ** -8) + p * dp_err

    def shared(x):
        return x.unflatten(1, (-1, g)).sum(2)

    n = p.shape[-1] + p.shape[-2] * g  # terms of the longest fp32 sums
    acc = n * 2.0 ** -24
    dv, dv_b = shared(p.transpose(2, 3) @ do), shared((p_err + acc * p).transpose(2, 3) @ do.abs())
    dk, dk_b = shared(ds.transpose(2, 3) @ q) * sm_scale, shared((ds_err + acc * ds.abs()).transpose(2, 3) @ q.abs()) * sm_scale
    dq, dq_b = ds @ kx * sm_scale, (ds_err + acc * ds.abs()) @ kx.abs() * sm_scale
    outs = []
    for x, b in ((dq, dq_b), (dk, dk_b), (dv, dv_b)):
        b = b + x.abs() * 2.0 ** -8 + 2.0 ** -133
        outs.append((x, b) if layout == "bhsd" else (x.transpose(1, 2), b.transpose(1, 2)))
    return outs


def make(b, hq, hkv, sq, skv, d, layout, seed=0, q_scale=1.0):
    gen = torch.Generator().manual_seed(seed)

    def t(h, s):
        return torch.randn((b, h, s, d) if layout == "bhsd" else (b, s, h, d), generator=gen)

    q, k, v, do = t(hq, sq) * q_scale, t(hkv, skv), t(hkv, skv), t(hq, sq)
    return [x.to(torch.bfloat16).cuda() for x in (q, k, v, do)]


def check(b, hq, hkv, sq, skv, d, causal, layout, seed=0, scale=None, q_scale=1.0):
    q, k, v, do = make(b, hq, hkv, sq, skv, d, layout, seed, q_scale)
    scale = d ** -0.5 if scale is None else scale
    o, lse = fa2.kernel_fn(q, k, v, causal, scale, layout=layout, return_lse=True)
    got = bwd.kernel_fn(do, q, k, v, o, lse, causal, scale, layout=layout)
    bwd.check_device_status(q.device)
    worst = []
    for name, x, (ref, bound) in zip(("dq", "dk", "dv"), got, formula(do, q, k, v, o, lse, causal, scale, layout)):
        assert x.shape == ref.shape and x.dtype == torch.bfloat16 and x.is_contiguous()
        used = ((x.double() - ref).abs() / bound).max().item()
        worst.append((name, used))
    assert all(w <= 1.0 for _, w in worst), worst


CASES = [
    # b, hq, hkv, sq, skv, d, causal, layout
    (1, 1, 1, 128, 128, 128, False, "bhsd"),
    (1, 1, 1, 128, 128, 128, True, "bhsd"),
    (1, 1, 1, 256, 256, 128, True, "bhsd"),
    (1, 1, 1, 64, 64, 256, True, "bhsd"),
    (1, 1, 1, 128, 128, 64, True, "bhsd"),
    (1, 2, 2, 1, 1, 128, True, "bhsd"),
    (1, 2, 1, 1, 1, 256, True, "bshd"),
    (1, 2, 2, 1, 1, 64, False, "bshd"),
    (1, 4, 2, 129, 129, 128, True, "bhsd"),
    (2, 4, 4, 257, 257, 128, True, "bhsd"),
    (1, 4, 2, 200, 200, 64, True, "bshd"),
    (1, 2, 1, 100, 100, 128, False, "bhsd"),
    (1, 8, 8, 512, 512, 64, True, "bshd"),
    (1, 4, 4, 1031, 1031, 128, True, "bhsd"),
    (2, 6, 3, 300, 300, 128, True, "bshd"),
    (1, 3, 1, 256, 256, 128, True, "bhsd"),
    (1, 10, 2, 333, 333, 64, False, "bhsd"),
    (3, 4, 1, 333, 333, 256, True, "bhsd"),
    (2, 8, 1, 200, 200, 256, True, "bshd"),
    (1, 2, 2, 65, 65, 256, False, "bhsd"),
    (1, 2, 2, 70, 500, 128, False, "bhsd"),    # more keys than queries
    (1, 2, 2, 500, 70, 128, False, "bshd"),    # more queries than keys
    (1, 2, 2, 70, 500, 128, True, "bhsd"),     # keys that no query sees
    (1, 2, 1, 500, 70, 64, True, "bhsd"),      # causal, queries behind the last key
    (1, 2, 1, 500, 70, 256, True, "bshd"),
    (1, 2, 1, 70, 500, 256, True, "bshd"),
    (1, 1, 1, 1, 1000, 128, False, "bhsd"),    # one query
    (1, 1, 1, 1000, 1, 64, False, "bhsd"),     # one key
]


@pytest.mark.parametrize("b,hq,hkv,sq,skv,d,causal,layout", CASES)
def test_gradients_match_the_formula(cuda_device, b, hq, hkv, sq, skv, d, causal, layout):
    check(b, hq, hkv, sq, skv, d, causal, layout, seed=sq + skv + hq)
